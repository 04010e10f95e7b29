"""8-bit linears: token quantization and the scaled integer product against
plain 64-bit implementations.

Tolerances: the codes and scales are exact.  The product's sum is exact; its
conversion to fp32, the token scale and the fused channel scale and bias round
once each (2^-24 relative to the scaled sum, or to the result), the output type
once more (half its spacing)."""

import ctypes
import os

import pytest
import torch

from g2ptq_b200 import _lib, ops
from g2ptq_b200.utils import int8_utils, moe_utils

gpu = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def built():
    from g2ptq_b200 import build
    if not (os.path.exists(_lib.LIB_PATH) and os.path.exists(build.BINDING)):
        build.build()


DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -24  # half the relative spacing of fp32


# -- plain 64-bit forms -------------------------------------------------------

def plain_quantize(x):
    v = x.double()
    top = v.abs().amax(1)
    finite = torch.isfinite(v).all(1)
    scale = (torch.where(finite, top, torch.zeros_like(top)) / 127).float()
    scale = torch.where(scale < torch.finfo(torch.float32).tiny, torch.ones_like(scale), scale)
    q = torch.round(torch.where(finite[:, None], v, torch.zeros_like(v)) / scale.double()[:, None])
    return q.to(torch.int8), torch.where(finite, scale, torch.full_like(scale, float("nan")))


def rounded(x, dtype):
    """Bound of the rounding of values of size |x| to dtype (its spacing below
    the normal range included)."""
    fi = torch.finfo(dtype)
    return x.abs() * (fi.eps / 2) + fi.tiny * fi.eps / 2


def check_product(got, a, sa, b, sb, bias):
    acc = a.double() @ b.double().T
    part = acc * sa.double()[:, None] * sb.double()
    want = part if bias is None else part + bias.double()
    tol = 2.01 * U * part.abs() + 1.01 * U * want.abs()
    # results past the type's largest value plus half its spacing there round to
    # infinity (fp16: 65504 + 16), results short of it do not
    fi = torch.finfo(got.dtype)
    edge = fi.max * (1 + fi.eps / 4)
    inf = torch.isinf(got) & (torch.sign(got.double()) == torch.sign(want))
    assert bool(inf[want.abs() - tol >= edge].all())
    assert not bool(torch.isinf(got)[want.abs() + tol < edge].any())
    tol = tol + rounded(want.abs() + tol, got.dtype)
    assert got.shape == want.shape
    assert bool((((got.double() - want).abs() <= tol) | inf).all())


def codes_of(shape, g, lo=-128):
    return torch.randint(lo, 128, shape, generator=g, device=DEV, dtype=torch.int8)


def aligned(codes):
    """The same codes with rows on 16-byte boundaries."""
    return int8_utils._int8_rows(codes)[..., :codes.shape[-1]]


def aligned_codes(shape, g):
    return aligned(codes_of(shape, g))


def gen(seed=0):
    return torch.Generator(device=DEV).manual_seed(seed)


# -- CPU: refusals ------------------------------------------------------------

def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.quantize_tokens(torch.zeros(2, 4))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.int8_matmul(torch.zeros(2, 4, dtype=torch.int8), torch.ones(2),
                        torch.zeros(3, 4, dtype=torch.int8), torch.ones(3))


def test_abi_refuses_bad_arguments():
    lib = _lib.load()
    p = ctypes.c_void_p(256)  # never dereferenced: the sizes are refused on the host
    bad = _lib.G2Q_ERR_INVALID_ARG
    assert lib.g2q_quantize_tokens(None, 16, None, None, 0, 16, 1, 16, None) == bad
    assert lib.g2q_quantize_tokens(p, 16, p, p, 7, 16, 1, 16, None) == bad
    assert lib.g2q_quantize_tokens(p, 8, p, p, 0, 16, 1, 16, None) == bad
    assert lib.g2q_quantize_tokens(None, 16, None, None, 0, 16, 0, 16, None) == 0
    args = [p, 0, 8, p, 16, p, p, 16, p, None]
    assert lib.g2q_int8_matmul(*args, 4, 8, 0, None, 0, None, None) == bad
    assert lib.g2q_int8_matmul(*args, 4, 9, 16, None, 0, None, None) == bad  # ldo < N
    assert lib.g2q_int8_matmul(*args, 4, 8, 17, None, 0, None, None) == bad  # lda < K
    args[4] = args[7] = 1 << 20
    assert lib.g2q_int8_matmul(*args, 4, 8, ops.INT8_MAX_K + 1, None, 0, None,
                               None) == _lib.G2Q_ERR_UNSUPPORTED
    assert lib.g2q_int8_matmul(None, 0, 8, None, 16, None, None, 16, None, None, 0, 8, 16, None, 0,
                               None, None) == 0
    assert lib.g2q_int8_matmul_grouped(p, 0, 8, p, 16, p, p, 16, 128, p, None, 2, 4, 8, 16, None,
                                       None) == bad
    assert lib.g2q_int8_matmul_grouped(p, 0, 8, p, 16, p, p, 16, 128, p, p, 1025, 4, 8, 16, None,
                                       None) == _lib.G2Q_ERR_UNSUPPORTED
    assert lib.g2q_int8_matmul_grouped(p, 0, 8, p, 16, p, p, 16, 127, p, p, 2, 4, 8, 16, None,
                                       None) == bad  # experts overlap


def test_quantizer_kinds_are_refused():
    from g2ptq_b200.utils.quant_utils import WeightQuantizer
    q = WeightQuantizer()
    q.configure(8, perchannel=True, sym=False)
    q._ready = True
    with pytest.raises(ValueError, match="symmetric"):
        int8_utils.weight_codes(torch.zeros(2, 4), q)
    q.configure(8, perchannel=True, sym=True, weight_groupsize=2)
    q._ready = True
    with pytest.raises(ValueError, match="groups"):
        int8_utils.weight_codes(torch.zeros(2, 4), q)


@pytest.mark.parametrize("M,K", [(17, 4100), (64, 4100), (200, 2050), (1000, 4100), (200, 4090),
                                 (4096, 8200)])
@pytest.mark.parametrize("G", [0, 1])
def test_one_channel_workspace(M, K, G):
    """The stride of a single channel does not decide whether its rows are aligned, so
    neither answer may leave out what the product's ranges of K need."""
    lib = _lib.load()
    codes = -(-M * ops.int8_row_stride(K) // 256) * 256 + -(-4 * M // 256) * 256
    product = lib.g2q_int8_matmul_workspace_bytes(M, 1, K) if G == 0 else 0
    assert G == 1 or K < 4000 or product > 0
    for aligned in (0, 1):
        assert lib.g2q_int8_linear_workspace_bytes(M, 1, K, G, aligned) >= codes + product


def test_lost_gradients_are_refused():
    """Nothing records a gradient here: an input that requires one is refused, not
    detached without a word."""
    import torch.autograd.forward_ad as fwad
    i8 = torch.zeros(3, 4, dtype=torch.int8)
    one, three = torch.ones(2), torch.ones(3)
    off = torch.tensor([0, 2], dtype=torch.int32)
    x = torch.ones(2, 4)

    def grad(t):
        return t.clone().requires_grad_()

    module = int8_utils.Int8Linear(i8, three)
    experts = int8_utils.Int8Experts(i8[None], three[None])
    calls = [lambda f: int8_utils.int8_linear(f(x), i8, three),
             lambda f: int8_utils.int8_linear(f(x[None]), i8, three),
             lambda f: int8_utils.int8_linear(x, i8, f(three)),
             lambda f: int8_utils.int8_linear(x, i8, three, f(three)),
             lambda f: int8_utils.int8_experts(f(x), i8[None], three[None], off),
             lambda f: int8_utils.int8_experts(x, i8[None], f(three[None]), off),
             lambda f: module(f(x)), lambda f: experts(f(x), off),
             lambda f: ops.int8_matmul(i8[:2], f(one), i8, three),
             lambda f: ops.int8_matmul_grouped(i8[:2], one, i8[None], f(three[None]), off)]
    for call in calls:
        with pytest.raises(RuntimeError, match="no gradient"):
            call(grad)
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
            call(grad)
        with fwad.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
            call(lambda t: fwad.make_dual(t, torch.ones_like(t)))


def test_experts_from_what_they_cannot_hold(monkeypatch):
    """A bias, or a linear without its quantizer, is refused instead of left out."""
    monkeypatch.setattr(int8_utils, "weight_codes",
                        lambda w, q: (torch.zeros(w.shape, dtype=torch.int8), torch.ones(len(w))))
    plain = [torch.nn.Linear(8, 4, bias=False) for _ in range(3)]
    assert int8_utils.Int8Experts.from_linears(plain, [None] * 3).codes.shape == (3, 4, 8)
    m = int8_utils.Int8Experts.from_linears((lin for lin in plain), iter([None] * 3))
    assert m.codes.shape == (3, 4, 8)
    with pytest.raises(ValueError, match="bias"):
        int8_utils.Int8Experts.from_linears(plain[:2] + [torch.nn.Linear(8, 4)], [None] * 3)
    for short in (plain[:2], plain + plain):
        with pytest.raises(ValueError):
            int8_utils.Int8Experts.from_linears(short, [None] * 3)


def test_rows_that_overlap_are_laid_out(monkeypatch):
    """A broadcast token, or windows over one, reach the product as plain rows."""
    seen = []
    monkeypatch.setattr(ops, "int8_linear", lambda x, *a: seen.append(x) or x[:, :1])
    monkeypatch.setattr(ops, "int8_linear_grouped", lambda x, *a: seen.append(x) or x[:, :1])
    row = torch.arange(8.0)
    for x in (row.expand(5, 8), row.expand(2, 3, 8), row.unfold(0, 4, 1), row[::2].expand(3, 4),
              torch.ones(4, 1).expand(4, 8), row.reshape(8, 1)[:1].expand(6, 1)):
        int8_utils.int8_linear(x, None, None)
        if x.dim() == 2:
            int8_utils.int8_experts(x, None, None, None)
        for got in seen:
            assert got.stride(0) >= got.shape[1] and got.stride(1) == 1
            assert torch.equal(got, x.reshape(-1, x.shape[-1]))
        seen.clear()
    plain = torch.ones(5, 16)[:, 4:12]
    int8_utils.int8_linear(plain, None, None)
    assert seen[0] is plain  # rows apart are no copy


CONVERSIONS = [lambda m: m.to(torch.bfloat16), lambda m: m.half(), lambda m: m.double(),
               lambda m: m.float(), lambda m: m.bfloat16().float(), lambda m: m.type(torch.float16)]


def converted(make, device):
    """Each conversion of a model that holds the module, and the module before it."""
    for convert in CONVERSIONS:
        mod = make()
        model = torch.nn.Sequential(torch.nn.Linear(3, 2), mod)
        before = {k: v.clone() for k, v in mod.state_dict().items()}
        convert(model.to(device))
        yield mod, before


def test_conversions_keep_codes_and_scales():
    rows, scale = torch.arange(-50, 50, dtype=torch.int8).reshape(5, 20), torch.rand(5) * 1e-3
    for make in (lambda: int8_utils.Int8Linear(rows, scale, torch.rand(5)),
                 lambda: int8_utils.Int8Linear(rows, scale),
                 lambda: int8_utils.Int8Experts(rows[None], scale[None])):
        for mod, before in converted(make, "cpu"):
            after = mod.state_dict()
            assert sorted(after) == sorted(before)
            for name, value in before.items():
                assert after[name].dtype == value.dtype and torch.equal(after[name], value)


# -- GPU: refusals ------------------------------------------------------------

@gpu
def test_refusals():
    i8 = lambda *s: torch.zeros(*s, dtype=torch.int8, device=DEV)  # noqa: E731
    f = lambda *s: torch.ones(*s, device=DEV)  # noqa: E731
    off = torch.zeros(3, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        ops.quantize_tokens(f(4))
    with pytest.raises(ValueError):
        ops.quantize_tokens(f(8, 4).t())
    with pytest.raises(ValueError):
        ops.quantize_tokens(f(1, 4).expand(3, 4))
    with pytest.raises(ValueError):
        ops.quantize_tokens(f(3, 0))
    with pytest.raises(TypeError):
        ops.quantize_tokens(f(3, 4).double())
    with pytest.raises(TypeError):
        ops.int8_matmul(f(2, 4), f(2), i8(3, 4), f(3))
    with pytest.raises(ValueError):
        ops.int8_matmul(i8(2, 4), f(2), i8(3, 5), f(3))
    with pytest.raises(ValueError):
        ops.int8_matmul(i8(2, 4), f(3), i8(3, 4), f(3))
    with pytest.raises(ValueError):
        ops.int8_matmul(i8(2, 4), f(2), i8(3, 4), f(3), bias=f(2))
    with pytest.raises(TypeError):
        ops.int8_matmul(i8(2, 4), f(2), i8(3, 4), f(3), out_dtype=torch.float64)
    with pytest.raises(ValueError):
        ops.int8_matmul_grouped(i8(2, 4), f(2), i8(3, 4), f(3), off)
    with pytest.raises(ValueError):
        ops.int8_matmul_grouped(i8(2, 4), f(2), i8(3, 5, 4), f(3, 5), off)
    with pytest.raises(ValueError):
        ops.int8_matmul_grouped(i8(2, 4), f(2), i8(2, 5, 4), f(2, 5), off.long())
    with pytest.raises(ValueError):
        ops.int8_matmul_grouped(i8(2, 4), f(2), i8(1, 5, 4).expand(2, 5, 4), f(2, 5), off)


@gpu
def test_library_errors_reach_the_caller():
    # more row tiles of unaligned operands than a grid has: refused before any launch
    a = torch.zeros(65536 * 64, 3, dtype=torch.int8, device=DEV)
    with pytest.raises(_lib.G2QError, match="unsupported"):
        ops.int8_matmul(a, torch.ones(a.shape[0], device=DEV),
                        torch.zeros(2, 3, dtype=torch.int8, device=DEV), torch.ones(2, device=DEV))


# -- quantization -------------------------------------------------------------

@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,C", [(1, 1), (3, 15), (1, 16), (5, 17), (700, 33), (1, 4096),
                                 (300, 1024), (301, 1040), (333, 8192), (2, 14336), (310, 9001),
                                 (2, 40000)])
def test_quantize_tokens(dtype, T, C):
    x = (torch.randn(T, C, generator=gen(T + C), device=DEV) * 3).to(dtype)
    x[:, 0] *= 20
    q, s = ops.quantize_tokens(x)
    wq, ws = plain_quantize(x)
    assert torch.equal(s, ws)
    assert torch.equal(q, wq)
    assert q.stride(0) % 16 == 0 or T == 1


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_ties_are_exact(dtype):
    # scale 1 or a power of two: every quotient is a multiple of 1/4, ties to even
    row = torch.cat([torch.arange(-507, 508, device=DEV) / 4.0, torch.tensor([127.0], device=DEV)])
    x = torch.stack([row, row * 2.0 ** -9, row * 2.0 ** 5]).to(dtype)
    q, s = ops.quantize_tokens(x)
    assert torch.equal(s, torch.tensor([1.0, 2.0 ** -9, 2.0 ** 5], device=DEV))
    wq, _ = plain_quantize(x)
    assert torch.equal(q, wq)


@gpu
def test_quantize_near_ties():
    # fp32 values next to half-integer multiples of a scale that is no power of two
    g = gen(3)
    scale = (torch.rand(400, 1, generator=g, device=DEV) + 0.5) * 1e-3
    top = scale * 127
    h = torch.randint(-126, 126, (400, 600), generator=g, device=DEV) + 0.5
    s = (top.double() / 127).float()
    x = (h.double() * s.double()).float()
    step = torch.randint(-2, 3, x.shape, generator=g, device=DEV, dtype=torch.int32)
    x = (x.view(torch.int32) + step).view(torch.float32)
    x = torch.cat([top, x], 1)
    q, got = ops.quantize_tokens(x)
    wq, ws = plain_quantize(x)
    assert torch.equal(got, ws) and torch.equal(q, wq)


@gpu
def test_quantize_near_ties_of_the_smallest_scales():
    """Quotients half a unit of the smallest fp32 number beside a half-integer: their
    distance from it, 2^-150, is no fp32 number itself."""
    unit = 2.0 ** -149
    steps = torch.arange(200, dtype=torch.int64)
    top = (127 * (2 ** 23 + 1000 + 9973 * steps)).double() * unit  # scales from 2^-126 up
    scale = (top.float().double() / 127).float()
    size = (scale.double() / unit).long()  # in units
    odd = size % 2 == 1
    assert int(odd.sum()) > 50 and bool((size[odd] < 2 ** 24 * 2 // 3).all())
    size, top = size[odd], top[odd].float()
    v = torch.stack([(size + 1) // 2, (size - 1) // 2, (3 * size + 1) // 2, (3 * size - 1) // 2], 1)
    x = torch.cat([top[:, None], (v.double() * unit).float(), (-v.double() * unit).float()], 1)
    # by whole numbers: round(v / size) lies where 2 v does beside the odd multiples of size
    want = torch.tensor([[127, 1, 0, 2, 1, -1, 0, -2, -1]]).expand(len(x), 9).to(torch.int8)
    q, s = plain_quantize(x)
    assert torch.equal(q, want)
    for rep in (1, 400 // len(x) + 1):  # few rows and many
        got, gs = ops.quantize_tokens(x.to(DEV).repeat(rep, 1))
        assert torch.equal(gs.cpu(), s.repeat(rep))
        assert torch.equal(got.cpu(), want.repeat(rep, 1))
    one = ops.int8_linear(x[:1].to(DEV), torch.eye(9, dtype=torch.int8, device=DEV),
                          torch.full((9,), 2.0 ** 126, device=DEV))  # in the product's own kernel
    assert torch.equal(torch.round(one.cpu().double() / (s[0].double() * 2.0 ** 126)),
                       want[:1].double())


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("C", [24, 1500, 20000])
def test_quantize_odd_rows(dtype, C):
    x = torch.randn(6, C, generator=gen(C), device=DEV).to(dtype)
    x[0] = 0
    x[1, C // 2] = float("inf")
    x[2, C - 1] = float("-inf")
    x[3, 0] = float("nan")
    x[4] = torch.finfo(dtype).max
    x[4, 1::2] *= -1
    q, s = ops.quantize_tokens(x)
    wq, ws = plain_quantize(x)
    assert torch.equal(q, wq)
    assert torch.equal(s.isnan(), ws.isnan()) and torch.equal(s[~s.isnan()], ws[~ws.isnan()])
    assert float(s[0]) == 1.0 and bool(s[1:4].isnan().all())


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pad,first", [(0, 0), (8, 0), (24, 8), (1, 0), (3, 1)])
def test_quantize_strides(dtype, pad, first):
    buf = torch.randn(37, 200 + pad + first, generator=gen(pad), device=DEV).to(dtype)
    x = buf[:, first:first + 200]
    q, s = ops.quantize_tokens(x)
    wq, ws = plain_quantize(x)
    assert torch.equal(q, wq) and torch.equal(s, ws)


# -- product ------------------------------------------------------------------

SHAPES = [(1, 1, 1), (1, 64, 16), (1, 1000, 4096), (7, 130, 100), (16, 257, 144), (17, 96, 512),
          (33, 520, 1040), (64, 128, 128), (100, 256, 2048), (129, 300, 272), (255, 256, 256),
          (256, 512, 384), (257, 1376, 512), (700, 1000, 1008), (1, 8, 20000), (1, 8000, 1040),
          (8, 100, 1024), (5, 9000, 500), (12, 70, 1000), (16, 48, 4112), (2, 40, 5000)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_int8_matmul(dtype, M, N, K):
    g = gen(M * 7 + N + K)
    a, b = aligned_codes((M, K), g), aligned_codes((N, K), g)
    sa = torch.rand(M, generator=g, device=DEV) * 1e-2
    sb = torch.rand(N, generator=g, device=DEV) * 1e-3
    for bias in (None, torch.randn(N, generator=g, device=DEV)):
        check_product(ops.int8_matmul(a, sa, b, sb, bias, out_dtype=dtype), a, sa, b, sb, bias)


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("M,N,K", [(9001, 5016, 2048), (8500, 5001, 2064), (9472, 4864, 2176)])
def test_int8_matmul_large(dtype, M, N, K):
    """Sizes at which the largest tiles are chosen, rows ending in each of a tile's
    blocks."""
    g = gen(M)
    a, b = aligned_codes((M, K), g), aligned_codes((N, K), g)
    sa, sb = torch.rand(M, generator=g, device=DEV), torch.rand(N, generator=g, device=DEV)
    check_product(ops.int8_matmul(a, sa, b, sb, out_dtype=dtype), a, sa, b, sb, None)


@gpu
@pytest.mark.parametrize("K", [2048, 2064])
@pytest.mark.parametrize("counts,tail", [([1100, 0, 613], 5), ([512, 1024, 257, 300], 0),
                                         ([3, 2000, 10], 700)])
def test_int8_matmul_grouped_large(counts, tail, K):
    a, sa, b, sb, off = grouped_case(counts, tail, 520, K, tail)
    got = ops.int8_matmul_grouped(a, sa, b, sb, off)
    cut = off.tolist()
    for e in range(len(counts)):
        lo, hi = cut[e], cut[e + 1]
        if hi > lo:
            check_product(got[lo:hi], a[lo:hi], sa[lo:hi], b[e], sb[e], None)
    assert not bool(got[cut[-1]:].any())


@gpu
@pytest.mark.parametrize("M,N,K,pa,pb", [(5, 70, 33, 0, 0), (70, 65, 130, 3, 1), (3, 9, 4, 0, 5),
                                         (130, 140, 63, 1, 0)])
def test_int8_matmul_unaligned_rows(M, N, K, pa, pb):
    g = gen(K)
    a, b = codes_of((M, K + pa), g)[:, :K], codes_of((N, K + pb), g)[:, :K]
    sa, sb = torch.rand(M, generator=g, device=DEV), torch.rand(N, generator=g, device=DEV)
    check_product(ops.int8_matmul(a, sa, b, sb), a, sa, b, sb, None)


@gpu
@pytest.mark.parametrize("M", [1, 40, 300])
def test_int8_matmul_extreme_codes(M):
    # the largest sums: every product 128 * 128 or -128 * 127
    K = ops.INT8_MAX_K - 15
    a = aligned(torch.full((M, K), -128, dtype=torch.int8, device=DEV))
    b = aligned(torch.full((3, K), -128, dtype=torch.int8, device=DEV))
    b[1] = 127
    sa, sb = torch.ones(M, device=DEV), torch.ones(3, device=DEV)
    check_product(ops.int8_matmul(a, sa, b, sb, out_dtype=torch.float32), a, sa, b, sb, None)


@gpu
def test_int8_matmul_nan_and_inf_scales():
    g = gen(1)
    a, b = aligned_codes((20, 64), g), aligned_codes((40, 64), g)
    sa, sb = torch.ones(20, device=DEV), torch.ones(40, device=DEV)
    sa[3] = float("nan")
    sb[5] = float("inf")
    got = ops.int8_matmul(a, sa, b, sb, out_dtype=torch.float32)
    want = (a.double() @ b.double().T) * sa.double()[:, None] * sb.double()
    assert torch.equal(got.isnan(), want.isnan())
    ok = ~want.isnan()
    assert torch.equal(got[ok].double(), want[ok])  # scales are 1: exact below 2^24


@gpu
def test_int8_matmul_empty():
    z = torch.zeros(0, 32, dtype=torch.int8, device=DEV)
    w = torch.zeros(5, 32, dtype=torch.int8, device=DEV)
    assert ops.int8_matmul(z, torch.ones(0, device=DEV), w, torch.ones(5, device=DEV)).shape == (0, 5)
    q, s = ops.quantize_tokens(torch.zeros(0, 32, device=DEV))
    assert q.shape == (0, 32) and s.shape == (0,)


def grouped_case(counts, tail, N, K, seed):
    g = gen(seed)
    E, R = len(counts), sum(counts) + tail
    a, b = aligned_codes((R, K), g), aligned_codes((E, N, K), g)
    sa = torch.rand(R, generator=g, device=DEV)
    sb = torch.rand(E, N, generator=g, device=DEV)
    off = torch.zeros(E + 1, dtype=torch.int32, device=DEV)
    off[1:] = torch.tensor(counts, device=DEV).cumsum(0)
    return a, sa, b, sb, off


COUNTS = [([0], 0), ([0, 0], 5), ([1], 0), ([3, 0, 0, 1], 2), ([16, 17, 15, 0, 33], 0),
          ([0, 300, 1, 129, 255], 7), ([256, 512, 0, 257], 300), ([2] * 60, 0),
          ([0] * 500 + [4] + [0] * 523, 1)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts,tail", COUNTS)
@pytest.mark.parametrize("N,K", [(130, 48), (300, 520)])
def test_int8_matmul_grouped(dtype, counts, tail, N, K):
    if len(counts) > 100:
        N = 20
    a, sa, b, sb, off = grouped_case(counts, tail, N, K, len(counts) + tail)
    got = ops.int8_matmul_grouped(a, sa, b, sb, off, out_dtype=dtype)
    cut = off.tolist()
    for e in range(len(counts)):
        lo, hi = cut[e], cut[e + 1]
        if hi > lo:
            check_product(got[lo:hi], a[lo:hi], sa[lo:hi], b[e], sb[e], None)
    assert not bool(got[cut[-1]:].any())


@gpu
@pytest.mark.parametrize("bad", ["descending", "beyond", "negative"])
def test_grouped_offsets_stay_in_bounds(bad):
    # offsets a caller got wrong: every row that is read or written exists; rows
    # of the ranges that are in order come out right
    a, sa, b, sb, off = grouped_case([10, 20, 30], 0, 40, 64, 5)
    if bad == "descending":
        off[2] = 5
    elif bad == "beyond":
        off[3] = 1 << 30
    else:
        off[1] = -(1 << 30)
    got = ops.int8_matmul_grouped(a, sa, b, sb, off)
    torch.cuda.synchronize()
    assert got.shape == (60, 40)
    if bad == "beyond":
        check_product(got[30:], a[30:], sa[30:], b[2], sb[2], None)


def partition(off, M):
    """The rows of each group, and behind the last, as the running maximum of the
    offsets within [0, M] cuts them."""
    cut, top = [0], 0
    for v in off[1:]:
        top = max(top, min(v, M))
        cut.append(top)
    return cut + [M]


BAD_OFFSETS = {
    "descending": lambda o, n: o[:n // 2] + [o[n // 2] // 3] + o[n // 2 + 1:],
    "saw": lambda o, n: [v if i % 2 else v // 2 for i, v in enumerate(o)],
    "negative": lambda o, n: o[:n // 3] + [-5] + o[n // 3 + 1:],
    "first": lambda o, n: [o[n // 2]] + o[1:],
    "beyond": lambda o, n: o[:-1] + [o[-1] + 1000],
    "all beyond": lambda o, n: [0] + [2 ** 31 - 1] * (len(o) - 1),
    "all negative": lambda o, n: [-2 ** 31] * len(o),
    "falling": lambda o, n: o[::-1],
}


@gpu
@pytest.mark.parametrize("bad", sorted(BAD_OFFSETS))
# few rows per group (the streaming kernel), many, and rows off 16-byte boundaries
@pytest.mark.parametrize("R,E,K", [(60, 40, 64), (500, 300, 64), (60, 3, 64), (700, 3, 64),
                                   (60, 40, 50), (3, 2, 64)])
def test_any_offsets_partition_the_rows(bad, R, E, K):
    g = gen(R + E)
    ids = torch.randint(0, E, (R - 2,), generator=g, device=DEV)
    good = [0] + torch.bincount(ids, minlength=E).cumsum(0).tolist()
    off = BAD_OFFSETS[bad](good, E)
    a, b = codes_of((R, K), g), codes_of((E, 24, K), g)
    a, b = (aligned(a), aligned(b)) if K % 16 == 0 else (a, b)
    sa, sb = torch.rand(R, generator=g, device=DEV), torch.rand(E, 24, generator=g, device=DEV)
    poison = torch.full((R, 24), float("nan"), device=DEV)  # what an unwritten row would show
    del poison
    got = ops.int8_matmul_grouped(a, sa, b, sb, torch.tensor(off, dtype=torch.int32, device=DEV),
                                  out_dtype=torch.float32)
    cut = partition(off, R)
    for e in range(E):
        lo, hi = cut[e], cut[e + 1]
        if hi > lo:
            check_product(got[lo:hi], a[lo:hi], sa[lo:hi], b[e], sb[e], None)
    assert not bool((got[cut[E]:] != 0).any())


@gpu
def test_grouped_strided_experts():
    g = gen(9)
    store = codes_of((4, 100, 128), g)
    b = store[:, 10:60, :96]
    a = aligned_codes((50, 96), g)
    sa, sb = torch.rand(50, generator=g, device=DEV), torch.rand(4, 50, generator=g, device=DEV)
    off = torch.tensor([0, 10, 10, 45, 50], dtype=torch.int32, device=DEV)
    got = ops.int8_matmul_grouped(a, sa, b, sb, off)
    for e, (lo, hi) in enumerate(((0, 10), (10, 10), (10, 45), (45, 50))):
        if hi > lo:
            check_product(got[lo:hi], a[lo:hi], sa[lo:hi], b[e], sb[e], None)


# -- the entry points together ------------------------------------------------

def linear_want(x, codes, scale, bias):
    q, s = plain_quantize(x)
    return q, s, codes, scale, bias


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,N", [((1, 512), 1376), ((2, 9, 130), 64), ((500, 272), 300),
                                     ((0, 64), 10), ((3, 0, 64), 10)])
def test_int8_linear(dtype, shape, N):
    g = gen(N)
    x = torch.randn(*shape, generator=g, device=DEV).to(dtype)
    codes = aligned_codes((N, shape[-1]), g)
    scale = torch.rand(N, generator=g, device=DEV) * 1e-2
    bias = torch.randn(N, generator=g, device=DEV)
    y = int8_utils.int8_linear(x, codes, scale, bias)
    assert y.shape == (*shape[:-1], N) and y.dtype == dtype
    if y.numel():
        q, s = plain_quantize(x.reshape(-1, shape[-1]))
        check_product(y.reshape(-1, N), q, s, codes, scale, bias)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts,tail", COUNTS)
def test_int8_experts(dtype, counts, tail):
    """One call for quantization and grouped product: the two calls' result."""
    g = gen(tail)
    a, _, b, sb, off = grouped_case(counts, tail, 40, 272, 77)
    x = torch.randn(a.shape, generator=g, device=DEV).to(dtype)
    got = int8_utils.int8_experts(x, b, sb, off)
    q, s = ops.quantize_tokens(x)
    assert torch.equal(got, ops.int8_matmul_grouped(q, s, b, sb, off, out_dtype=dtype))


@gpu
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_int8_linear_is_its_two_steps(M, N, K):
    g = gen(M + N + K)
    x = torch.randn(M, K, generator=g, device=DEV)
    b, sb = aligned_codes((N, K), g), torch.rand(N, generator=g, device=DEV)
    q, s = ops.quantize_tokens(x)
    want = ops.int8_matmul(q, s, b, sb, out_dtype=x.dtype)
    for _ in range(20):  # back to back: the product overlaps the quantization's end
        got = int8_utils.int8_linear(x, b, sb)
    assert torch.equal(got, want)
    assert torch.equal(ops.int8_linear(x, b.contiguous(), sb), want)  # rows of any alignment


@gpu
@pytest.mark.parametrize("M,N,K", [(8, 4096, 4096), (3, 300, 20000), (16, 512, 2064), (64, 520, 1040),
                                   (200, 512, 14336), (700, 1000, 1008)])
def test_int8_linear_of_changing_inputs(M, N, K):
    """Back to back calls whose inputs differ and whose workspace is the same memory:
    every product reads its own call's codes and scales, not what the call before
    left there while the quantization was still writing."""
    g = gen(M + N)
    b, sb = aligned_codes((N, K), g), torch.rand(N, generator=g, device=DEV)
    xs = [torch.randn(M, K, generator=g, device=DEV) * 2.0 ** (i % 5) for i in range(12)]
    pairs = [ops.quantize_tokens(x) for x in xs]
    want = [ops.int8_matmul(q, s, b, sb, out_dtype=torch.float32) for q, s in pairs]
    torch.cuda.synchronize()
    got = [int8_utils.int8_linear(x, b, sb) for x in xs]
    for a, w in zip(got, want):
        assert torch.equal(a, w)


@gpu
@pytest.mark.parametrize("R,E", [(32, 128), (900, 4)])
def test_int8_experts_of_changing_inputs(R, E):
    g = gen(R)
    N, K = 200, 2048
    b, sb = aligned_codes((E, N, K), g), torch.rand(E, N, generator=g, device=DEV)
    off = torch.zeros(E + 1, dtype=torch.int32, device=DEV)
    off[1:] = torch.bincount(torch.randint(0, E, (R - 3,), generator=g, device=DEV),
                             minlength=E).cumsum(0)  # three rows without an expert
    xs = [torch.randn(R, K, generator=g, device=DEV) * 2.0 ** (i % 5) for i in range(12)]
    pairs = [ops.quantize_tokens(x) for x in xs]
    want = [ops.int8_matmul_grouped(q, s, b, sb, off, out_dtype=torch.float32) for q, s in pairs]
    torch.cuda.synchronize()
    got = [int8_utils.int8_experts(x, b, sb, off) for x in xs]
    for a, w in zip(got, want):
        assert torch.equal(a, w) and not bool(a[-3:].any())


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 4100), (5, 4100), (17, 4100), (64, 1666), (64, 4100),
                                 (200, 2050), (200, 4096), (1000, 4100), (4096, 8200)])
def test_int8_linear_one_channel(dtype, M, K):
    """One output channel, its row's stride anything: K itself, or what a view has."""
    g = gen(M + K)
    x = torch.randn(M, K, generator=g, device=DEV).to(dtype)
    codes, scale = codes_of((1, K), g), torch.rand(1, generator=g, device=DEV)
    bias = torch.randn(1, generator=g, device=DEV)
    q, s = plain_quantize(x)
    wide = torch.zeros(1, K + 5, dtype=torch.int8, device=DEV)
    wide[:, :K] = codes
    for c in (codes, aligned(codes), wide[:, :K]):
        check_product(int8_utils.int8_linear(x, c, scale, bias), q, s, codes, scale, bias)
    check_product(int8_utils.Int8Linear(codes, scale)(x), q, s, codes, scale, None)
    off = torch.tensor([0, M], dtype=torch.int32, device=DEV)
    check_product(int8_utils.int8_experts(x, codes[None], scale[None], off), q, s, codes, scale,
                  None)


@gpu
def test_int8_linear_refusals():
    w, s = torch.zeros(3, 4, dtype=torch.int8, device=DEV), torch.ones(3, device=DEV)
    x = torch.zeros(2, 4, device=DEV)
    off = torch.zeros(2, dtype=torch.int32, device=DEV)
    for bad in (lambda: ops.int8_linear(x[:, :3], w, s), lambda: ops.int8_linear(x, w, s[:2]),
                lambda: ops.int8_linear(x[0], w, s), lambda: ops.int8_linear(x, w, s.half()),
                lambda: ops.int8_linear(x, w, s, x[0]),
                lambda: ops.int8_linear_grouped(x, w, s, off),
                lambda: ops.int8_linear_grouped(x, w[None], s[None], off[:1])):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: ops.int8_linear(x, w.float(), s), lambda: ops.int8_linear(x.double(), w, s),
                lambda: ops.int8_linear_grouped(x.double(), w[None], s[None], off)):
        with pytest.raises(TypeError):
            bad()


@gpu
def test_int8_linear_transposed_input():
    g = gen(4)
    x = torch.randn(64, 30, generator=g, device=DEV).t()
    codes, scale = aligned_codes((50, 64), g), torch.ones(50, device=DEV)
    q, s = plain_quantize(x)
    check_product(int8_utils.int8_linear(x, codes, scale), q, s, codes, scale, None)


@gpu
def test_int8_linear_broadcast_input():
    g = gen(5)
    codes, scale = aligned_codes((50, 64), g), torch.ones(50, device=DEV)
    off = torch.tensor([0, 7], dtype=torch.int32, device=DEV)
    row = torch.randn(64, generator=g, device=DEV)
    for x in (row.expand(7, 64), torch.randn(70, generator=g, device=DEV).unfold(0, 64, 1)):
        q, s = plain_quantize(x)
        check_product(int8_utils.int8_linear(x, codes, scale), q, s, codes, scale, None)
        check_product(int8_utils.int8_experts(x, codes[None], scale[None], off), q, s, codes,
                      scale, None)
    y = int8_utils.int8_linear(row.expand(2, 3, 64), codes, scale)
    q, s = plain_quantize(row.expand(6, 64))
    check_product(y.reshape(6, 50), q, s, codes, scale, None)


@gpu
def test_linear_from_a_quantized_weight():
    """GPTQ with an 8-bit symmetric per-channel quantizer, then the 8-bit linear on
    its codes: they reproduce the quantized weight."""
    from g2ptq_b200.gptq_utils import gptq_utils
    from g2ptq_b200.gptq_utils.common_utils import make_group_quantizers
    from g2ptq_b200.utils.quant_utils import WeightQuantizer
    g = gen(11)
    lin = torch.nn.Linear(256, 192, bias=True, device=DEV)
    lin.weight.data = torch.randn(192, 256, generator=g, device=DEV) * 0.02
    x = torch.randn(4, 128, 256, generator=g, device=DEV)
    obj = gptq_utils.GPTQ([lin])
    quantizer = WeightQuantizer()
    quantizer.configure(8, perchannel=True, sym=True)
    obj.quantizer = make_group_quantizers(quantizer, 256, -1)
    obj.add_batch(0, x, None)
    obj.fasterquant(blocksize=128, percdamp=0.01, groupsize=-1, actorder=False, static_groups=False)
    m = int8_utils.Int8Linear.from_linear(lin, obj.quantizer[0])
    back = m.codes.double() * m.scale.double()[:, None]
    w = lin.weight.data.double()
    assert bool(((back - w).abs() <= U * w.abs() + 1e-30).all())
    q, s = plain_quantize(x.reshape(-1, 256))
    check_product(m(x).reshape(-1, 192), q, s, m.codes, m.scale, lin.bias.data)


@gpu
@pytest.mark.parametrize("K", [96, 100])
def test_modules_keep_their_layout(K):
    """Copies, moves and state dicts of a module keep rows that the tensor cores
    take, and its results."""
    import copy
    g = gen(K)
    m = int8_utils.Int8Linear(codes_of((70, K), g), torch.rand(70, generator=g, device=DEV),
                              torch.randn(70, generator=g, device=DEV))
    x = torch.randn(50, K, generator=g, device=DEV)
    want = m(x)
    other = int8_utils.Int8Linear(codes_of((70, K), g), torch.rand(70, generator=g, device=DEV),
                                  torch.zeros(70, device=DEV))
    other.load_state_dict(m.state_dict())
    for mod in (copy.deepcopy(m), copy.deepcopy(m).cpu().to(DEV), other):
        assert mod.codes.shape == (70, K) and mod.codes.stride(0) % 16 == 0
        assert torch.equal(mod.codes, m.codes) and torch.equal(mod(x), want)
    e = int8_utils.Int8Experts(codes_of((3, 20, K), g), torch.ones(3, 20, device=DEV))
    assert e.codes.shape == (3, 20, K) and e.codes.stride(1) % 16 == 0


@gpu
def test_converted_modules_give_the_same():
    g = gen(3)
    codes, scale = codes_of((70, 100), g), torch.rand(70, generator=g, device=DEV) * 1e-2
    bias = torch.randn(70, generator=g, device=DEV)
    x = torch.randn(50, 100, generator=g, device=DEV).to(torch.bfloat16)
    off = torch.tensor([0, 50], dtype=torch.int32, device=DEV)
    want = int8_utils.Int8Linear(codes, scale, bias)(x)
    for mod, _ in converted(lambda: int8_utils.Int8Linear(codes.cpu(), scale.cpu(), bias.cpu()), DEV):
        assert torch.equal(mod(x), want) and mod.codes.stride(0) % 16 == 0
    want = int8_utils.Int8Experts(codes[None], scale[None])(x, off)
    for mod, _ in converted(lambda: int8_utils.Int8Experts(codes[None].cpu(), scale[None].cpu()),
                            DEV):
        assert torch.equal(mod(x, off), want)


@gpu
def test_side_stream_and_graph():
    g = gen(6)
    codes, scale = aligned_codes((300, 512), g), torch.rand(300, generator=g, device=DEV)
    x = torch.randn(70, 512, generator=g, device=DEV).to(torch.bfloat16)
    want = int8_utils.int8_linear(x, codes, scale)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = int8_utils.int8_linear(x, codes, scale)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    # two graphs of the same weight, replayed at once on two streams
    graphs, outs, ins = [], [], []
    for k in range(2):
        xi = x.clone()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            y = int8_utils.int8_linear(xi, codes, scale)
        graphs.append(gr)
        ins.append(xi)
        outs.append(y)
    fresh = [torch.randn(70, 512, generator=g, device=DEV).to(torch.bfloat16) for _ in range(2)]
    for xi, f in zip(ins, fresh):
        xi.copy_(f)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for gr, st in zip(graphs, streams):
        with torch.cuda.stream(st):
            for _ in range(3):
                gr.replay()
    torch.cuda.synchronize()
    for y, f in zip(outs, fresh):
        assert torch.equal(y, int8_utils.int8_linear(f, codes, scale))


@gpu
def test_capture_without_a_status_word():
    """A first call inside a capture makes no status word there: its zeros would be
    written by a replay only."""
    g = gen(8)
    codes, scale = aligned_codes((64, 128), g), torch.rand(64, generator=g, device=DEV)
    x = torch.randn(300, 128, generator=g, device=DEV)
    want = int8_utils.int8_linear(x, codes, scale)  # loads the library
    words = dict(ops._DEVICE_STATUS)
    ops._DEVICE_STATUS.clear()
    try:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            y = int8_utils.int8_linear(x, codes, scale)
        assert not ops._DEVICE_STATUS
    finally:
        ops._DEVICE_STATUS.update(words)
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, want)


@gpu
def test_moe_layer_in_8_bits():
    """Router, sort, gate / up and down of every expert in 8 bits and the weighted
    way back, against the same steps in 64 bits on the same codes."""
    g = gen(21)
    T, E, k, H, I = 50, 6, 2, 128, 96
    x = torch.randn(T, H, generator=g, device=DEV)
    top, ids = torch.topk(torch.randn(T, E, generator=g, device=DEV), k, dim=-1)
    w = torch.softmax(top, -1)
    ids[0] = -1  # a token without any expert
    gu = int8_utils.Int8Experts(codes_of((E, 2 * I, H), g),
                                torch.rand(E, 2 * I, generator=g, device=DEV) * 2e-3)
    down = int8_utils.Int8Experts(codes_of((E, H, I), g),
                                  torch.rand(E, H, generator=g, device=DEV) * 2e-3)
    r = moe_utils.route(ids, E)
    rows = moe_utils.dispatch(x, r)
    h = gu(rows, r.offsets)
    act = torch.nn.functional.silu(h[:, :I]) * h[:, I:]
    out = moe_utils.combine(down(act, r.offsets), r, w)
    want = torch.zeros(T, H, dtype=torch.float64, device=DEV)
    bound = torch.zeros_like(want)
    cut = r.offsets.tolist()
    q2, s2 = plain_quantize(act)  # of the same activations: what is tested is the routing and products
    for e in range(E):
        for row in range(cut[e], cut[e + 1]):
            pair = int(r.order[row])
            t, j = divmod(pair, k)
            q1, s1 = plain_quantize(x[t:t + 1])
            check_product(h[row:row + 1], q1, s1, gu.codes[e], gu.scale[e], None)
            y = (q2[row].double() @ down.codes[e].double().T) * s2[row].double() * down.scale[e].double()
            want[t] += w[t, j].double() * y
            bound[t] += (w[t, j].double() * y).abs()
    # 3 roundings in the product, one per fused multiply-add, one to fp32
    assert bool(((out.double() - want).abs() <= (3 + k + 1) * 1.01 * U * bound).all())
    assert not bool(out[0].any())
