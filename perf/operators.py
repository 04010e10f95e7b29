"""The 8-bit product and expert-routing operators as cases to measure.

``run`` computes each operator either in its plain form (elementary torch
operations) or, where ``own`` is true, through the package's entry points:

* ``linear``   -- a quantized linear: every token of ``x`` gets its own scale
  (largest magnitude / 127) and int8 codes, the codes are multiplied with the
  int8 weight codes, and the product is scaled per token and per channel;
* ``experts``  -- the same for rows sorted by expert, each range of rows with
  its own expert's weight;
* ``dispatch`` -- the (token, slot) pairs of a top-k routing sorted by expert
  (stable) and the tokens' rows copied into that order; with ``grad`` also the
  gradient of the tokens;
* ``combine``  -- the experts' rows brought back to the tokens' order, weighted
  and summed; with ``grad`` also the gradients of the rows and of the weights.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # one token through a 4096 x 4096 projection: the latency of decoding
        dict(name="linear_decode_one", op="linear", tokens=1, rows=4096, cols=4096,
             dtype="bf16", bias=False, pad=0),
        # a decoding batch through the up projection: streaming the weight
        dict(name="linear_decode_batch", op="linear", tokens=24, rows=14336, cols=4096,
             dtype="bf16", bias=False, pad=0),
        # a short prompt through the down projection, long sums
        dict(name="linear_prompt_down", op="linear", tokens=200, rows=4096, cols=14336,
             dtype="fp16", bias=False, pad=8),
        # the CPU-sized block's MLP in fp32 with a bias and an odd token count
        dict(name="linear_small_fp32_bias", op="linear", tokens=511, rows=1376, cols=512,
             dtype="fp32", bias=True, pad=0),
        # a forward batch of 8 calibration sequences through the up projection
        dict(name="linear_calibration", op="linear", tokens=16384, rows=14336, cols=4096,
             dtype="bf16", bias=False, pad=0),
        # four decoded tokens through gate and up of 128 experts
        dict(name="experts_decode", op="experts", tokens=4, topk=8, experts=128, rows=1536,
             cols=2048, dtype="bf16", drop=0.0),
        # a calibration batch through the 128 experts' down projections
        dict(name="experts_calibration", op="experts", tokens=8192, topk=8, experts=128,
             rows=2048, cols=768, dtype="bf16", drop=0.0),
        # a decoding batch sorted by expert
        dict(name="dispatch_decode", op="dispatch", tokens=16, topk=8, experts=128, cols=2048,
             dtype="bf16", drop=0.0, grad=False),
        # a forward batch of 32 calibration sequences sorted by expert
        dict(name="dispatch_calibration", op="dispatch", tokens=65536, topk=8, experts=128,
             cols=2048, dtype="bf16", drop=0.0, grad=False),
        # a refresh step's routing with the tokens' gradient, ragged sizes, some
        # slots routed to experts of another process
        dict(name="dispatch_refresh_odd", op="dispatch", tokens=3001, topk=2, experts=9,
             cols=1376, dtype="fp32", drop=0.2, grad=True),
        # a decoding batch back in token order
        dict(name="combine_decode", op="combine", tokens=33, topk=8, experts=128, cols=2048,
             dtype="bf16", drop=0.0, grad=False),
        # a refresh step's batch back in token order, with both gradients
        dict(name="combine_refresh", op="combine", tokens=16384, topk=8, experts=128, cols=2048,
             dtype="bf16", drop=0.0, grad=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "experts", "dispatch", "combine"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "linear":
        tokens, rows, cols = _log(rng, 1, 16384), _log(rng, 64, 14336), _log(rng, 64, 14336)
        cols = min(cols, 16384 * 14336 * 4096 // (tokens * rows))
        return dict(op=op, tokens=tokens, rows=rows, cols=cols, dtype=dtype,
                    bias=rng.random() < 0.3, pad=rng.choice([0, 0, 8, 24]))
    experts = _log(rng, 2, 128)
    topk = rng.randint(1, min(8, experts))
    drop = rng.choice([0.0, 0.0, 0.1])
    if op == "experts":
        tokens, rows, cols = _log(rng, 1, 8192), _log(rng, 64, 2048), _log(rng, 64, 2048)
        tokens = max(1, min(tokens, 65536 * 768 // (topk * cols)))
        return dict(op=op, tokens=tokens, topk=topk, experts=experts, rows=rows, cols=cols,
                    dtype=dtype, drop=drop)
    cols = _log(rng, 64, 4096)
    most = 65536 * 8 * 2048 * 2 if op == "dispatch" else 16384 * 8 * 2048 * 2
    grad = rng.random() < 0.5
    most //= 4 if grad and op == "dispatch" else 1
    tokens = max(1, min(_log(rng, 1, 65536), most // (topk * cols * BYTES[dtype])))
    return dict(op=op, tokens=tokens, topk=topk, experts=experts, cols=cols, dtype=dtype,
                drop=drop, grad=grad)


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------

def _hidden(tokens, cols, dtype, g, pad=0):
    """Hidden states N(0, 1) with a few channels 20 times larger, rows ``cols + pad`` apart."""
    x = torch.randn(tokens, cols + pad, device="cuda", generator=g)
    loud = torch.randint(0, cols, (4,), device="cuda", generator=g)
    x[:, loud] *= 20.0
    return x.to(DTYPES[dtype])[:, :cols]


def _weight(shape, g):
    """int8 codes and channel scales of weights N(0, 0.02), rows on 16-byte boundaries
    (laid out once, when the weight is quantized)."""
    *lead, cols = shape
    ld = -(-cols // 16) * 16
    codes = torch.zeros(*lead, ld, dtype=torch.int8, device="cuda")[..., :cols]
    codes.copy_((torch.randn(*shape, device="cuda", generator=g) * 32).round_().clamp_(-128, 127))
    scale = (torch.rand(*lead, device="cuda", generator=g) + 0.5) * (0.02 / 32)
    return codes, scale


def _routing(case, g):
    """Top-k experts of a router with a skewed load and their softmax weights; ``drop``:
    the share of slots whose expert lives elsewhere (id -1)."""
    T, E, k = case["tokens"], case["experts"], case["topk"]
    logits = torch.randn(T, E, device="cuda", generator=g)
    logits += 0.7 * torch.randn(E, device="cuda", generator=g)
    top, ids = torch.topk(logits, k, dim=-1)
    weights = torch.softmax(top, dim=-1)
    if case["drop"]:
        away = torch.rand(T, k, device="cuda", generator=g) < case["drop"]
        ids = torch.where(away, torch.full_like(ids, -1), ids)
    return ids, weights


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(case=case)
    if case["op"] == "linear":
        st["x"] = _hidden(case["tokens"], case["cols"], case["dtype"], g, case["pad"])
        st["codes"], st["scale"] = _weight((case["rows"], case["cols"]), g)
        st["bias"] = (torch.randn(case["rows"], device="cuda", generator=g)
                      if case["bias"] else None)
        return st
    ids, weights = _routing(case, g)
    n = ids.numel()
    if case["op"] == "dispatch":
        st["ids"] = ids
        st["x"] = _hidden(case["tokens"], case["cols"], case["dtype"], g)
        if case["grad"]:
            st["g"] = torch.randn(n, case["cols"], device="cuda", generator=g).to(
                DTYPES[case["dtype"]])
        return st
    order, position, offsets = _plain_route(ids, case["experts"])
    if case["op"] == "experts":
        st["offsets"] = offsets
        st["x"] = _hidden(n, case["cols"], case["dtype"], g)
        st["codes"], st["scale"] = _weight((case["experts"], case["rows"], case["cols"]), g)
        return st
    st.update(order=order, position=position, offsets=offsets, w=weights)
    st["y"] = torch.randn(n, case["cols"], device="cuda", generator=g).to(DTYPES[case["dtype"]])
    if case["grad"]:
        st["g"] = torch.randn(case["tokens"], case["cols"], device="cuda", generator=g).to(
            DTYPES[case["dtype"]])
    return st


# --------------------------------------------------------------------------
# the plain forms
# --------------------------------------------------------------------------

def _plain_quantize(x):
    """Scales fp32(max |x| / 127) and codes round(x / scale), ties to even; the quotient in
    64 bits, since a 32-bit one can fall on the other side of a tie."""
    xf = x.float()
    scale = (xf.abs().amax(-1).double() / 127).float()
    return torch.round(xf.double() / scale.double()[:, None]).float(), scale


def _plain_linear(st):
    q, s = _plain_quantize(st["x"])
    y = (q @ st["codes"].float().T) * s[:, None] * st["scale"]
    if st["bias"] is not None:
        y = y + st["bias"]
    return y.to(st["x"].dtype)


def _plain_experts(st):
    """Each expert's rows padded to the longest range, one batched product; rows behind
    the last range give zeros."""
    x, off = st["x"], st["offsets"].long()
    n, E = x.shape[0], off.numel() - 1
    q, s = _plain_quantize(x)
    row = torch.arange(n, device=x.device)
    expert = torch.searchsorted(off[1:].contiguous(), row, right=True)
    used = expert < E
    e = expert.clamp(max=E - 1)
    cap = max(1, int((off[1:] - off[:-1]).max()))
    slot = torch.where(used, row - off[e], torch.full_like(row, cap))
    padded = torch.zeros(E, cap + 1, x.shape[1], device=x.device)
    padded[e, slot] = q
    y = torch.bmm(padded, st["codes"].float().transpose(1, 2))[e, slot]
    y = y * s[:, None] * st["scale"][e]
    return torch.where(used[:, None], y, torch.zeros_like(y)).to(x.dtype)


def _plain_route(ids, E):
    """``order``: the pairs token * k + slot in expert order (stable); ``position [T, k]``:
    each pair's row there; ``offsets [E + 1]``: each expert's rows.  Pairs whose id is
    no expert come last, their position p given as -1 - p."""
    flat = ids.reshape(-1)
    valid = (flat >= 0) & (flat < E)
    key = torch.where(valid, flat, torch.full_like(flat, E))
    order = torch.argsort(key, stable=True)
    position = torch.empty_like(order)
    position[order] = torch.arange(order.numel(), device=order.device)
    position = torch.where(valid, position, -1 - position)
    edges = torch.arange(E + 1, device=ids.device)
    offsets = torch.searchsorted(key[order], edges)
    return order.int(), position.int().reshape(ids.shape), offsets.int()


def _plain_dispatch(st):
    x, E, k = st["x"], st["case"]["experts"], st["case"]["topk"]
    order, position, offsets = _plain_route(st["ids"], E)
    rows = x[order.long() // k]
    used = torch.arange(rows.shape[0], device=x.device) < offsets[-1]
    rows = torch.where(used[:, None], rows, torch.zeros_like(rows))
    out = dict(rows=rows, order=order, position=position, offsets=offsets)
    if st["case"]["grad"]:
        p = position.long()
        part = st["g"][p.clamp(min=0)].float() * (p >= 0).float()[..., None]
        out["grad_x"] = part.sum(1).to(x.dtype)
    return out


def _plain_combine(st):
    y, p, w = st["y"], st["position"].long(), st["w"]
    live = p >= 0
    yf = y[p.clamp(min=0)].float()
    wl = torch.where(live, w, torch.zeros_like(w))
    out = dict(out=(yf * wl[..., None]).sum(1).to(y.dtype))
    if st["case"]["grad"]:
        g = st["g"].float()
        row = torch.where(live, p, -1 - p)
        grad_y = torch.empty_like(y)
        grad_y[row.reshape(-1)] = (wl[..., None] * g[:, None]).to(y.dtype).flatten(0, 1)
        out["grad_y"] = grad_y
        out["grad_w"] = torch.where(live, (yf * g[:, None]).sum(-1), torch.zeros_like(w))
    return out


PLAIN = dict(linear=_plain_linear, experts=_plain_experts, dispatch=_plain_dispatch,
             combine=_plain_combine)


# --------------------------------------------------------------------------
# the package's calls
# --------------------------------------------------------------------------

def _own_run(st):
    from g2ptq_b200.utils import int8_utils, moe_utils
    op = st["case"]["op"]
    if op == "linear":
        return int8_utils.int8_linear(st["x"], st["codes"], st["scale"], st["bias"])
    if op == "experts":
        return int8_utils.int8_experts(st["x"], st["codes"], st["scale"], st["offsets"])
    grad = st["case"]["grad"]
    if op == "dispatch":
        x = st["x"].detach().requires_grad_() if grad else st["x"]
        r = moe_utils.route(st["ids"], st["case"]["experts"])
        rows = moe_utils.dispatch(x, r)
        out = dict(rows=rows.detach(), order=r.order, position=r.position, offsets=r.offsets)
        if grad:
            (out["grad_x"],) = torch.autograd.grad(rows, x, st["g"])
        return out
    r = moe_utils.Routing(st["order"], st["position"], st["offsets"])
    if not grad:
        return dict(out=moe_utils.combine(st["y"], r, st["w"]))
    y, w = st["y"].detach().requires_grad_(), st["w"].detach().requires_grad_()
    o = moe_utils.combine(y, r, w)
    grad_y, grad_w = torch.autograd.grad(o, (y, w), st["g"])
    return dict(out=o.detach(), grad_y=grad_y, grad_w=grad_w)


def run(state):
    return _own_run(state) if own else PLAIN[state["case"]["op"]](state)


# --------------------------------------------------------------------------
# what a pass cannot do without, and its result in 64 bits
# --------------------------------------------------------------------------

def work(case):
    b = BYTES[case["dtype"]]
    T, C = case["tokens"], case["cols"]
    if case["op"] == "linear":
        R = case["rows"]
        return dict(bytes=T * C * b + R * C + 4 * R * (2 if case["bias"] else 1) + T * R * b,
                    flops=2 * T * R * C)
    n, E = T * case["topk"], case["experts"]
    live = n * (1 - case["drop"])
    if case["op"] == "experts":
        R = case["rows"]
        hit = E * (1 - (1 - case["topk"] * (1 - case["drop"]) / E) ** T)  # experts with rows
        return dict(bytes=live * C * b + n * R * b + hit * R * (C + 4) + 4 * (E + 1),
                    flops=2 * live * R * C)
    route = 8 * n + 4 * (2 * n + E + 1)
    if case["op"] == "dispatch":
        return dict(bytes=route + T * C * b + n * C * b
                    + ((live + T) * C * b if case["grad"] else 0),
                    flops=live * C if case["grad"] else n)
    fwd = live * C * b + T * C * b + 8 * n
    # the gradients' pass reads the rows and the output's gradient again
    bwd = (live + n + T) * C * b + 12 * n if case["grad"] else 0
    return dict(bytes=fwd + bwd, flops=live * C * (5 if case["grad"] else 2))


def _exact_codes(x):
    """The codes of each row and its scale, as 64-bit values."""
    v = x.to(torch.float64)
    top = v.abs().max(dim=1, keepdim=True).values
    scale = (top / 127.0).to(torch.float32).to(torch.float64)
    return (v / scale).round(), scale


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "linear":
        q, s = _exact_codes(st["x"])
        y = torch.mm(q, st["codes"].to(torch.float64).t())
        y.mul_(s).mul_(st["scale"].to(torch.float64)[None])
        return y if st["bias"] is None else y.add_(st["bias"].to(torch.float64)[None])
    if case["op"] == "experts":
        q, s = _exact_codes(st["x"])
        y = torch.zeros(q.shape[0], case["rows"], dtype=torch.float64, device="cuda")
        cut = st["offsets"].tolist()
        for e in range(case["experts"]):
            a, b = cut[e], cut[e + 1]
            if b > a:
                part = torch.mm(q[a:b], st["codes"][e].to(torch.float64).t())
                y[a:b] = part * s[a:b] * st["scale"][e].to(torch.float64)[None]
        return y
    T, k, C = case["tokens"], case["topk"], case["cols"]
    if case["op"] == "dispatch":
        ids = st["ids"].reshape(-1)
        token = torch.arange(T, device="cuda").repeat_interleave(k)
        slot_of = torch.full((T * k,), -1, dtype=torch.int64, device="cuda")
        rows = torch.zeros(T * k, C, dtype=torch.float64, device="cuda")
        at = 0
        for e in range(case["experts"]):
            pairs = torch.nonzero(ids == e).reshape(-1)
            slot_of[pairs] = torch.arange(at, at + pairs.numel(), device="cuda")
            rows[at:at + pairs.numel()] = st["x"][token[pairs]].to(torch.float64)
            at += pairs.numel()
        out = dict(rows=rows, order=None, position=None, offsets=None)
        if case["grad"]:
            gx = torch.zeros(T, C, dtype=torch.float64, device="cuda")
            here = slot_of >= 0
            gx.index_add_(0, token[here], st["g"].to(torch.float64)[slot_of[here]])
            out["grad_x"] = gx
        return out
    p, w = st["position"].to(torch.int64), st["w"].to(torch.float64)
    out = torch.zeros(T, C, dtype=torch.float64, device="cuda")
    grad_y = torch.zeros(T * k, C, dtype=torch.float64, device="cuda")
    grad_w = torch.zeros(T, k, dtype=torch.float64, device="cuda")
    for j in range(k):
        t = torch.nonzero(p[:, j] >= 0).reshape(-1)
        r = p[t, j]
        y = st["y"][r].to(torch.float64)
        out[t] += w[t, j, None] * y
        if case["grad"]:
            g = st["g"][t].to(torch.float64)
            grad_y[r] = w[t, j, None] * g
            grad_w[t, j] = torch.einsum("tc,tc->t", g, y)
    return dict(out=out, grad_y=grad_y, grad_w=grad_w) if case["grad"] else dict(out=out)
