"""Expert routing: the stable sort by expert, the copies there and back and
their gradients against plain 64-bit implementations.

Tolerances: the sort and the copies are exact.  A weighted sum of k rows rounds
once per fused multiply-add (2^-24 of the sum of magnitudes) and once to the
output's type; a dot product over C columns adds at most ceil(C / 32) + 25
terms in a chain (columns per lane, pieces of at most 16, the tree)."""

import ctypes
import os

import pytest
import torch

from g2ptq_b200 import _lib, ops
from g2ptq_b200.utils import moe_utils

gpu = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def built():
    from g2ptq_b200 import build
    if not (os.path.exists(_lib.LIB_PATH) and os.path.exists(build.BINDING)):
        build.build()


DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -24


def gen(seed=0):
    return torch.Generator(device=DEV).manual_seed(seed)


def plain_route(ids, E):
    flat = ids.reshape(-1).tolist()
    lists = [[] for _ in range(E + 1)]
    for i, e in enumerate(flat):
        lists[e if 0 <= e < E else E].append(i)
    order = [i for part in lists for i in part]
    offsets, at = [], 0
    for part in lists:
        offsets.append(at)
        at += len(part)
    position = [0] * len(flat)
    for r, i in enumerate(order):
        position[i] = r if r < offsets[E] else -1 - r
    return (torch.tensor(order, dtype=torch.int32), torch.tensor(position, dtype=torch.int32),
            torch.tensor(offsets, dtype=torch.int32))


def check_route(ids, E):
    r = moe_utils.route(ids, E)
    order, position, offsets = plain_route(ids.cpu(), E)
    assert torch.equal(r.order.cpu(), order)
    assert torch.equal(r.position.cpu().reshape(-1), position)
    assert torch.equal(r.offsets.cpu(), offsets)
    return r


def rounded(x, dtype):
    fi = torch.finfo(dtype)
    return x.abs() * (fi.eps / 2) + fi.tiny * fi.eps / 2


# -- CPU ----------------------------------------------------------------------

def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.route(torch.zeros(2, 2, dtype=torch.int64), 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.dispatch_rows(torch.zeros(2, 4), torch.zeros(2, 2, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.combine_rows(torch.zeros(4, 4), torch.zeros(2, 2, dtype=torch.int32))


def test_abi_refuses_bad_arguments():
    lib = _lib.load()
    p = ctypes.c_void_p(256)  # never dereferenced: refused on the host
    bad, uns = _lib.G2Q_ERR_INVALID_ARG, _lib.G2Q_ERR_UNSUPPORTED
    assert lib.g2q_route(p, p, None, p, 1, 4, 4, None, 0, None) == bad
    assert lib.g2q_route(p, p, p, p, 2, 4, 4, None, 0, None) == bad
    assert lib.g2q_route(p, p, p, p, 1, 4, 0, None, 0, None) == bad
    assert lib.g2q_route(p, p, p, p, 1, 4, 1025, None, 0, None) == uns
    assert lib.g2q_route(p, p, p, p, 1, 1 << 31, 4, p, 1 << 40, None) == uns
    assert lib.g2q_route(None, p, p, p, 1, 4, 4, None, 0, None) == bad
    need = lib.g2q_route_workspace_bytes(100000, 16)
    assert need > 0 and lib.g2q_route_workspace_bytes(100, 16) == 0
    assert lib.g2q_route(p, p, p, p, 1, 100000, 16, p, need - 1, None) == bad
    assert lib.g2q_dispatch_rows(p, 8, p, 8, 3, p, 2, 2, 8, None) == bad
    assert lib.g2q_dispatch_rows(p, 7, p, 8, 2, p, 2, 2, 8, None) == bad
    assert lib.g2q_dispatch_rows(p, 8, p, 8, 2, p, 1 << 30, 2, 8, None) == bad
    assert lib.g2q_dispatch_rows(None, 8, None, 8, 2, None, 0, 2, 8, None) == 0
    assert lib.g2q_combine_rows(p, 8, p, 8, 5, p, p, 1, 2, 2, 8, None) == bad
    assert lib.g2q_combine_rows(p, 8, p, 8, 0, p, p, 5, 2, 2, 8, None) == bad
    assert lib.g2q_combine_rows_backward(p, 8, p, p, 8, p, 8, 0, p, None, 1, 2, 2, 8, None) == bad
    assert lib.g2q_combine_rows_backward(p, 8, p, p, 8, None, 8, 0, p, p, 1, 2, 2, 8, None) == bad
    assert lib.g2q_combine_rows_backward(None, 0, None, p, 8, p, 8, 0, p, p, 1, 2, 2, 8, None) == 0


# -- GPU ----------------------------------------------------------------------

@gpu
def test_refusals():
    ids = torch.zeros(3, 2, dtype=torch.int64, device=DEV)
    r = moe_utils.route(ids, 4)
    x = torch.zeros(3, 8, device=DEV)
    y = torch.zeros(6, 8, device=DEV)
    w = torch.zeros(3, 2, device=DEV)
    for bad in (lambda: ops.route(ids[0], 4), lambda: ops.route(ids, 0),
                lambda: ops.route(ids, 1025), lambda: ops.route(ids.t(), 4),
                lambda: ops.dispatch_rows(x[:2], r.position),
                lambda: ops.dispatch_rows(x, r.position.long()),
                lambda: ops.dispatch_rows(x[:1].expand(3, 8), r.position),
                lambda: ops.combine_rows(y[:5], r.position, w),
                lambda: ops.combine_rows(y, r.position, w[:2]),
                lambda: ops.combine_rows_backward(x[:2], y, r.position, w),
                lambda: ops.combine_rows_backward(x.half(), y, r.position, w),
                lambda: ops.combine_rows_backward(x, y, r.position, None)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.route(ids.float(), 4), lambda: ops.dispatch_rows(x.double(), r.position),
                lambda: ops.combine_rows(y.double(), r.position, w),
                lambda: ops.combine_rows(y, r.position, w.double()),
                lambda: moe_utils.dispatch(x.double().requires_grad_(), r)):
        with pytest.raises(TypeError):
            bad()


@gpu
@pytest.mark.parametrize("T,k,E", [(0, 2, 4), (1, 1, 1), (1, 8, 128), (16, 8, 128), (33, 3, 5),
                                   (4096, 1, 7), (4097, 1, 7), (3001, 2, 9), (1000, 8, 1024),
                                   (20000, 8, 128), (90001, 7, 33)])
@pytest.mark.parametrize("wide", [True, False])
def test_route(T, k, E, wide):
    g = gen(T + k + E)
    ids = torch.randint(0, E, (T, k), generator=g, device=DEV)
    ids = ids if wide else ids.int()
    check_route(ids, E)


@gpu
def test_route_skew_drops_and_repeats():
    g = gen(1)
    ids = torch.randint(-2, 12, (5000, 3), generator=g, device=DEV)
    check_route(ids, 10)  # -2, -1, 10 and 11 are no experts
    check_route(torch.full((3000, 2), 4, device=DEV), 9)  # one expert takes all
    check_route(torch.full((3000, 2), -1, device=DEV), 9)  # none takes any
    check_route(torch.tensor([[2 ** 40, 1], [-2 ** 40, 1]], device=DEV), 3)


def check_dispatch(x, r):
    rows = moe_utils.dispatch(x, r)
    T, k = r.position.shape
    want = torch.zeros(T * k, x.shape[1], dtype=x.dtype, device=DEV)
    used = int(r.offsets[-1])
    want[:used] = x[r.order[:used].long() // k]
    assert rows.is_contiguous()
    assert torch.equal(rows.view(torch.uint8 if x.dtype == torch.int8 else x.dtype),
                       want.view(torch.uint8 if x.dtype == torch.int8 else x.dtype))


COLS = [1, 2, 7, 64, 73, 130, 1024, 1376, 2515, 4096]


@gpu
@pytest.mark.parametrize("dtype", DTYPES + [torch.int8])
@pytest.mark.parametrize("C", COLS)
def test_dispatch(dtype, C):
    g = gen(C)
    for T, k in ((1, 1), (5, 8), (301, 3)):
        ids = torch.randint(-1, 6, (T, k), generator=g, device=DEV)
        x = (torch.randn(T, C, generator=g, device=DEV) * 30).to(dtype)
        check_dispatch(x, check_route(ids, 6))


@gpu
@pytest.mark.parametrize("first,pad", [(0, 8), (8, 0), (1, 0), (3, 5)])
def test_dispatch_strides(first, pad):
    g = gen(first)
    buf = torch.randn(40, 96 + first + pad, generator=g, device=DEV).to(torch.bfloat16)
    ids = torch.randint(0, 4, (40, 2), generator=g, device=DEV)
    check_dispatch(buf[:, first:first + 96], check_route(ids, 4))


def check_combine(y, r, w):
    T, k = r.position.shape
    out = moe_utils.combine(y, r, w)
    p = r.position.long()
    live = (p >= 0).double()
    wd = live if w is None else w.double() * live
    part = y.double()[p.clamp(min=0)] * wd[..., None]
    part = torch.where(live[..., None] > 0, part, torch.zeros_like(part))
    want, size = part.sum(1), part.abs().sum(1)
    tol = k * 1.01 * U * size
    tol = tol + rounded(want.abs() + tol, y.dtype)
    assert out.dtype == y.dtype and bool(((out.double() - want).abs() <= tol).all())


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", COLS)
@pytest.mark.parametrize("T,k,w_dtype", [(1, 1, torch.float32), (5, 8, torch.bfloat16),
                                         (301, 3, torch.float16), (40, 19, torch.float32),
                                         (33, 4, None)])
def test_combine(dtype, C, T, k, w_dtype):
    g = gen(C + T)
    ids = torch.randint(-1, 6, (T, k), generator=g, device=DEV)
    ids[0] = -1  # a token without any expert
    r = moe_utils.route(ids, 6)
    y = torch.randn(T * k, C, generator=g, device=DEV).to(dtype)
    y[int(r.offsets[-1]):] = float("nan")  # rows that nothing may read
    w = None if w_dtype is None else torch.rand(T, k, generator=g, device=DEV).to(w_dtype)
    check_combine(y, r, w)
    assert not bool(moe_utils.combine(y, r, w)[0].any())


def plain_backward(g, y, r, w):
    """(grad_y, grad_w, the dot products' sums of magnitudes) in 64 bits."""
    p = r.position.long()
    live = p >= 0
    gd, wd = g.double(), torch.where(live, w.double(), torch.zeros_like(w.double()))
    gy = torch.zeros(y.shape, dtype=torch.float64, device=DEV)
    row = torch.where(live, p, -1 - p).reshape(-1)
    gy[row] = (wd[..., None] * gd[:, None]).flatten(0, 1)
    prod = y.double()[p.clamp(min=0)] * gd[:, None]
    prod = torch.where(live[..., None], prod, torch.zeros_like(prod))
    return gy, prod.sum(-1), prod.abs().sum(-1)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [1, 7, 64, 130, 513, 1376, 4096])
@pytest.mark.parametrize("T,k,w_dtype", [(1, 1, torch.float32), (5, 8, torch.bfloat16),
                                         (150, 3, torch.float32), (30, 11, torch.float16)])
def test_gradients(dtype, C, T, k, w_dtype):
    g = gen(C + T + k)
    ids = torch.randint(-1, 6, (T, k), generator=g, device=DEV)
    r = moe_utils.route(ids, 6)
    x = torch.randn(T, C, generator=g, device=DEV).to(dtype).requires_grad_()
    rows = moe_utils.dispatch(x, r)
    gr = torch.randn(T * k, C, generator=g, device=DEV).to(dtype)
    (gx,) = torch.autograd.grad(rows, x, gr)
    p = r.position.long()
    part = gr.double()[p.clamp(min=0)] * (p >= 0).double()[..., None]
    want, size = part.sum(1), part.abs().sum(1)
    tol = k * 1.01 * U * size
    assert bool(((gx.double() - want).abs() <= tol + rounded(want.abs() + tol, dtype)).all())

    y = torch.randn(T * k, C, generator=g, device=DEV).to(dtype).requires_grad_()
    w = torch.rand(T, k, generator=g, device=DEV).to(w_dtype).requires_grad_()
    go = torch.randn(T, C, generator=g, device=DEV).to(dtype)
    out = moe_utils.combine(y, r, w)
    gy, gw = torch.autograd.grad(out, (y, w), go)
    wy, ww, size = plain_backward(go, y.detach(), r, w.detach())
    tol = 1.01 * U * wy.abs()
    assert bool(((gy.double() - wy).abs() <= tol + rounded(wy.abs() + tol, dtype)).all())
    tol = (-(-C // 32) + 25) * 1.01 * U * size
    assert gw.dtype == w_dtype
    assert bool(((gw.double() - ww).abs() <= tol + rounded(ww.abs() + tol, w_dtype)).all())


@gpu
def test_gradients_against_differences():
    # combine is linear in the rows and in the weights: differences at step 1 are
    # exact up to the roundings of the two values they subtract
    g = gen(8)
    T, k, C = 21, 3, 77
    r = moe_utils.route(torch.randint(-1, 5, (T, k), generator=g, device=DEV), 5)
    y, dy = (torch.randn(T * k, C, generator=g, device=DEV) for _ in range(2))
    w, dw = (torch.randn(T, k, generator=g, device=DEV) for _ in range(2))
    go = torch.randn(T, C, generator=g, device=DEV)
    gy, gw = ops.combine_rows_backward(go, y, r.position, w)

    def value(yy, ww):
        return (ops.combine_rows(yy, r.position, ww).double() * go.double()).sum()

    size = T * C * k * 8.0 * 4.0  # magnitudes: k terms of |w| |y| (below 8 on average), times |g|
    num = (value(y + dy, w) - value(y - dy, w)) / 2
    ana = (gy.double() * dy.double()).sum()
    assert abs(float(num - ana)) <= (k + 4) * U * size
    num = (value(y, w + dw) - value(y, w - dw)) / 2
    ana = (gw.double() * dw.double()).sum()
    assert abs(float(num - ana)) <= (C / 32 + 25 + k + 4) * U * size


@gpu
def test_gradients_that_are_not_needed():
    g = gen(2)
    r = moe_utils.route(torch.randint(0, 4, (9, 2), generator=g, device=DEV), 4)
    y = torch.randn(18, 40, generator=g, device=DEV)
    w = torch.rand(9, 2, generator=g, device=DEV)
    go = torch.randn(9, 40, generator=g, device=DEV)
    gy, gw = ops.combine_rows_backward(go, y, r.position, w)
    y1 = y.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(moe_utils.combine(y1, r, w), y1, go)[0], gy)
    w1 = w.clone().requires_grad_()
    assert torch.equal(torch.autograd.grad(moe_utils.combine(y, r, w1), w1, go)[0], gw)
    # without weights, and a gradient that autograd broadcast (stride zero)
    y2 = y.clone().requires_grad_()
    moe_utils.combine(y2, r).sum().backward()
    assert torch.equal(y2.grad, torch.ones_like(y))
    with torch.no_grad():
        assert moe_utils.dispatch(go.requires_grad_(), r).grad_fn is None


def test_library_errors_keep_their_type():
    """A negative status of the library is a G2QError through the native binding too."""
    p = torch.zeros(2, 2, dtype=torch.int32)
    mod = _lib.binding()
    with pytest.raises(RuntimeError, match="CUDA"):
        mod.combine_rows(torch.zeros(4, 4), p, None)
    assert issubclass(_lib.G2QError, RuntimeError)


def test_forward_mode_is_refused():
    """A tangent that nothing carries on is refused, with and without a gradient."""
    import torch.autograd.forward_ad as fwad
    p = torch.zeros(2, 2, dtype=torch.int32)
    r = moe_utils.Routing(p.reshape(-1), p, p[0])
    x, y, w = torch.ones(2, 4), torch.ones(4, 4), torch.ones(2, 2)
    with fwad.dual_level():
        dual = lambda t: fwad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: moe_utils.dispatch(dual(x), r), lambda: moe_utils.combine(dual(y), r),
                     lambda: moe_utils.combine(dual(y), r, w),
                     lambda: moe_utils.combine(y, r, dual(w)),
                     lambda: moe_utils.dispatch(dual(x.clone().requires_grad_()), r)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_another_extension_of_the_same_short_name(tmp_path):
    """Some other package's extension called _binding is not this one."""
    import importlib.util
    import shutil
    from g2ptq_b200 import build
    mine = _lib.binding()
    path = str(tmp_path / "_binding.so")
    shutil.copy(build.BINDING, path)
    spec = importlib.util.spec_from_file_location("_binding", path)
    other = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(other)
    assert other is not mine and mine.__spec__.origin == build.BINDING


@gpu
def test_a_refused_size_is_a_library_error():
    # more elements per slot than the library indexes: refused before any launch
    lib = _lib.load()
    x = torch.zeros(2, 8, device=DEV)
    pos = torch.zeros(2, 2, dtype=torch.int32, device=DEV)
    assert lib.g2q_dispatch_rows(x.data_ptr(), 4, x.data_ptr(), 8, 4, pos.data_ptr(), 2, 2, 8,
                                 None) == _lib.G2Q_ERR_INVALID_ARG
    with pytest.raises(_lib.G2QError, match="invalid argument"):
        _lib.call("g2q_dispatch_rows", x.data_ptr(), 4, x.data_ptr(), 8, 4, pos.data_ptr(), 2, 2,
                  8, None)


def failing_binding(tmp_path, names, status):
    """A second copy of the binding, in which the library's functions `names` return
    `status` without doing anything."""
    import importlib.util
    import shutil
    from g2ptq_b200 import build
    path = str(tmp_path / "_binding.so")
    shutil.copy(build.BINDING, path)
    _lib.binding()  # torch and the library are loaded
    failing_binding.keep.append(path)
    spec = importlib.util.spec_from_file_location(
        f"failing{len(failing_binding.keep)}._binding", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    fail = ctypes.CFUNCTYPE(ctypes.c_int)(lambda: status)
    failing_binding.keep.append(fail)  # called by address, so never freed
    address = {n: ctypes.cast(getattr(_lib.load(), n), ctypes.c_void_p).value for n in _lib._BOUND}
    address.update({n: ctypes.cast(fail, ctypes.c_void_p).value for n in names})
    mod.bind(address, _lib.G2QError, lambda idx: 0)
    return mod


failing_binding.keep = []


@gpu
def test_errors_of_the_library_reach_the_caller(tmp_path):
    g = gen(6)
    ids = torch.randint(0, 4, (9, 2), generator=g, device=DEV)
    r = moe_utils.route(ids, 4)
    x, y = (torch.randn(n, 8, generator=g, device=DEV) for n in (9, 18))
    w = torch.rand(9, 2, generator=g, device=DEV)
    names = ("g2q_route", "g2q_dispatch_rows", "g2q_combine_rows", "g2q_combine_rows_backward")
    mod = failing_binding(tmp_path, names, _lib.G2Q_ERR_UNSUPPORTED)
    for name, call in zip(names, (
            lambda m: m.route(ids, 4), lambda m: m.dispatch_rows(x, r.position),
            lambda m: m.combine_rows(y, r.position, w),
            lambda m: m.combine_rows_backward(x, y, r.position, w, True, True))):
        with pytest.raises(_lib.G2QError, match=f"{name}.*unsupported") as e:
            call(mod)
        assert e.value.status == _lib.G2Q_ERR_UNSUPPORTED
        call(_lib.binding())
    for call in (lambda m: m.dispatch(x.clone().requires_grad_(), r.position),
                 lambda m: m.combine(y.clone().requires_grad_(), r.position, w)):
        with pytest.raises(_lib.G2QError):
            call(mod)
        assert call(_lib.binding()).requires_grad


@gpu
def test_errors_of_the_library_in_a_backward(tmp_path):
    """There the engine's thread has no interpreter to make a G2QError with: a plain
    error of the same text, and the process goes on."""
    g = gen(7)
    r = moe_utils.route(torch.randint(0, 4, (9, 2), generator=g, device=DEV), 4)
    y = torch.randn(18, 8, generator=g, device=DEV).requires_grad_()
    w = torch.rand(9, 2, generator=g, device=DEV).requires_grad_()
    mod = failing_binding(tmp_path, ("g2q_combine_rows_backward", "g2q_dispatch_rows"),
                          _lib.G2Q_ERR_INVALID_ARG)
    with pytest.raises(RuntimeError, match="g2q_combine_rows_backward failed: .*invalid argument"):
        mod.combine(y, r.position, w).sum().backward()
    with pytest.raises(RuntimeError, match="g2q_dispatch_rows failed: .*invalid argument"):
        mod.combine(y, r.position, None).sum().backward()
    assert y.grad is None and w.grad is None
    moe_utils.combine(y, r, w).sum().backward()
    gy, gw = ops.combine_rows_backward(torch.ones(9, 8, device=DEV), y.detach(), r.position,
                                       w.detach())
    assert torch.equal(y.grad, gy) and torch.equal(w.grad, gw)


@gpu
def test_second_derivatives_are_refused():
    g = gen(4)
    r = moe_utils.route(torch.randint(0, 4, (9, 2), generator=g, device=DEV), 4)
    x = torch.randn(9, 8, generator=g, device=DEV).requires_grad_()
    w = torch.rand(9, 2, generator=g, device=DEV).requires_grad_()
    out = moe_utils.combine(moe_utils.dispatch(x, r), r, w)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(out.sum(), x, create_graph=True)


@gpu
def test_rows_changed_in_place_are_noticed():
    g = gen(4)
    r = moe_utils.route(torch.randint(0, 4, (9, 2), generator=g, device=DEV), 4)
    y = torch.randn(18, 8, generator=g, device=DEV)
    w = torch.rand(9, 2, generator=g, device=DEV).requires_grad_()
    out = moe_utils.combine(y, r, w)
    y.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()


@gpu
def test_rows_beyond_32_bit_offsets():
    g = gen(5)
    T, k, C = 40000, 8, 8192  # 2.6e9 elements
    ids = torch.randint(0, 16, (T, k), generator=g, device=DEV)
    r = moe_utils.route(ids, 16)
    x = torch.randn(T, C, generator=g, device=DEV).to(torch.bfloat16)
    rows = moe_utils.dispatch(x, r)
    for i in range(0, T * k, T):
        at = r.order[i:i + T].long() // k
        assert torch.equal(rows[i:i + T], x[at])
    # k equal rows with weights 1/8 give the token back exactly
    w = torch.full((T, k), 0.125, device=DEV)
    assert torch.equal(moe_utils.combine(rows, r, w), x)
    gy, gw = ops.combine_rows_backward(x, rows, r.position, w)
    last = int(r.order[-1])
    assert torch.equal(gy[-1], x[last // k] * 0.125)
    want = (x[last // k].double() ** 2).sum()
    assert abs(float(gw.reshape(-1)[last].double() - want)) <= (C / 32 + 25) * 1.01 * U * float(want)


class Expert(torch.nn.Module):
    def __init__(self, H, I, dtype, g):
        super().__init__()
        self.up = torch.nn.Linear(H, I, bias=False, device=DEV, dtype=dtype)
        self.down = torch.nn.Linear(I, H, bias=False, device=DEV, dtype=dtype)
        for m in (self.up, self.down):
            m.weight.data.copy_(torch.randn(m.weight.shape, generator=g, device=DEV) * 0.1)

    def forward(self, x):
        return self.down(torch.relu(self.up(x)))


@gpu
def test_routed_experts_forward():
    """The routed forward and its backward against the loop over hit experts in
    64 bits; hooks see the routed tokens only; an unhit expert is not called."""
    g = gen(13)
    T, E, k, H, I = 60, 5, 2, 48, 64
    experts = [Expert(H, I, torch.float32, g) for _ in range(E)]
    seen = {}
    for e, ex in enumerate(experts):
        ex.up.register_forward_hook(
            lambda m, a, out, e=e: seen.update({e: a[0].detach().clone()}))
    x = torch.randn(T, H, generator=g, device=DEV).requires_grad_()
    ids = torch.randint(0, E - 1, (T, k), generator=g, device=DEV)  # the last expert is not hit
    ids[3] = -1
    w = torch.rand(T, k, generator=g, device=DEV).requires_grad_()
    go = torch.randn(T, H, generator=g, device=DEV)
    out = moe_utils.routed_experts_forward(experts, x, ids, w)
    gx, gw = torch.autograd.grad(out, (x, w), go)

    xd, wd = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
    want = torch.zeros(T, H, dtype=torch.float64, device=DEV)
    for e in range(E):
        tok, slot = torch.nonzero(ids == e, as_tuple=True)
        if tok.numel() == 0:
            continue
        h = torch.relu(xd[tok] @ experts[e].up.weight.double().T)
        y = h @ experts[e].down.weight.double().T
        want = want.index_add(0, tok, y * wd[tok, slot, None])
    wx, ww = torch.autograd.grad(want, (xd, wd), go.double())
    assert sorted(seen) == [e for e in range(E) if bool((ids == e).any())]
    for e, rows in seen.items():
        tok, _ = torch.nonzero(ids == e, as_tuple=True)
        assert torch.equal(rows, x.detach()[tok])
    # two chained fp32 products of lengths H and I (and their transposes): at most
    # (H + I + T) roundings of 2^-24 relative to sums of magnitudes, which stay
    # below 20 times the largest result here
    for got, ref in ((out.detach(), want.detach()), (gx, wx), (gw, ww)):
        assert float((got.double() - ref).abs().max()) <= (H + I + T) * U * 20 * float(ref.abs().max())


@gpu
def test_no_token_has_an_expert():
    g = gen(14)
    experts = [Expert(8, 8, torch.float32, g)]
    x = torch.randn(4, 8, generator=g, device=DEV).requires_grad_()
    w = torch.ones(4, 2, device=DEV).requires_grad_()
    out = moe_utils.routed_experts_forward(experts, x, torch.full((4, 2), -1, device=DEV), w)
    assert out.shape == x.shape and not bool(out.any())
    gx, gw = torch.autograd.grad(out.sum(), (x, w))
    assert not bool(gx.any()) and not bool(gw.any())


@gpu
def test_side_stream_and_graph_with_backward():
    g = gen(15)
    T, k, E, C = 70, 4, 8, 96
    ids = torch.randint(0, E, (T, k), generator=g, device=DEV)
    x = torch.randn(T, C, generator=g, device=DEV)
    w = torch.rand(T, k, generator=g, device=DEV)
    go = torch.randn(T, C, generator=g, device=DEV)

    def step(x, w, ids, go):
        r = moe_utils.route(ids, E)
        rows = moe_utils.dispatch(x, r)
        out = moe_utils.combine(rows, r, w)
        return (out.detach(), *torch.autograd.grad(out, (x, w), go))

    def leaves(x, w):
        return x.clone().requires_grad_(), w.clone().requires_grad_()

    want = step(*leaves(x, w), ids, go)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(*leaves(x, w), ids, go)
        sx, sw = leaves(x, w)  # warm-up of the captured leaves
        step(sx, sw, ids, go)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    sids, sgo = ids.clone(), go.clone()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        outs = step(sx, sw, sids, sgo)
    ids2 = torch.randint(-1, E, (T, k), generator=g, device=DEV)
    x2 = torch.randn(T, C, generator=g, device=DEV)
    with torch.no_grad():
        sids.copy_(ids2)
        sx.copy_(x2)
    gr.replay()
    torch.cuda.synchronize()
    want = step(*leaves(x2, w), ids2, go)
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
