"""Microscaled 4-bit expert weights and the router's balance loss, as cases to
time.

A case is a dict of plain values; `prepare` makes a program's tensors from a
seed, `run` is one pass through an operator: the framework's calls where `own`
is set, elementary torch operations in 32 bits where it is not.  `exact` is the
same result from the definitions in 64 bits.

    quantize     weights to e2m1 codes with a power-of-two scale per 32 of a
                 row, and back: what a converter runs and checks itself by
    gather       one expert projection: out[t, k] = x[t] @ W[idx[t, k]]^T
    experts      a SwiGLU expert bank: gate, up and down of every (t, k)
    balance      loss = E sum_e f_e P_e, f_e the share of the kept tokens'
                 choices that fell on expert e, P_e their mean probability of it
    balance_vjp  its gradient in the logits, plus that of the renormalised
                 top-k weights

Shapes are those of the configurations c2, c4, c5 and c6 (hidden size d,
experts E, choices K, expert width f).  Weights are N(0, 0.02), x is N(0, 1),
routing logits N(0, 1) over a per-expert N(0, 0.5).
"""
import math

import torch

own = False

# hidden size, experts, choices per token, expert width, most tokens of a call
SHAPES = {
    "c2": (2048, 128, 8, 768, 4096),
    "c4": (2048, 512, 10, 512, 2048),
    "c5": (4096, 128, 8, 1536, 512),
    "c6": (2048, 256, 8, 512, 2048),
}
GROUP = 32
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def listed():
    return [
        # converting a checkpoint: one expert bank, quantised and read back
        {"name": "quantize_c2_bank", "kind": "quantize", "experts": 128, "rows": 768,
         "cols": 2048, "f32": False},
        # one projection of a shared expert held in f32, a ragged slice of it
        {"name": "quantize_f32_509_rows", "kind": "quantize", "experts": 1, "rows": 509,
         "cols": 2080, "f32": True},
        # one token's expert projection: the latency of interactive decoding
        {"name": "gather_c2_up_T1", "kind": "gather", "cfg": "c2", "proj": "up", "tokens": 1},
        # an odd-sized chunk of a prompt through one down projection
        {"name": "gather_c6_down_T509", "kind": "gather", "cfg": "c6", "proj": "down",
         "tokens": 509},
        # a handful of sequences decoding together
        {"name": "experts_c6_T7", "kind": "experts", "cfg": "c6", "tokens": 7},
        # a serving batch: every expert's weights read for a few rows each
        {"name": "experts_c2_T64", "kind": "experts", "cfg": "c2", "tokens": 64},
        # a prompt chunk over many small experts
        {"name": "experts_c4_T2048", "kind": "experts", "cfg": "c4", "tokens": 2048},
        # a long prompt: the products bound it
        {"name": "experts_c2_T4096", "kind": "experts", "cfg": "c2", "tokens": 4096},
        # load statistics of a decode batch
        {"name": "balance_c2_T64", "kind": "balance", "tokens": 64, "experts": 128, "k": 8,
         "bf16": False, "mask": False},
        # one training micro-batch of padded sequences, many experts
        {"name": "balance_c4_T32768_mask", "kind": "balance", "tokens": 32768, "experts": 512,
         "k": 10, "bf16": False, "mask": True},
        # fine-tuning a bf16 router on a short padded batch
        {"name": "balance_vjp_c2_T1000_bf16", "kind": "balance_vjp", "tokens": 1000,
         "experts": 128, "k": 8, "bf16": True, "mask": True},
        # the backward pass of the large micro-batch
        {"name": "balance_vjp_c4_T32768", "kind": "balance_vjp", "tokens": 32768,
         "experts": 512, "k": 10, "bf16": False, "mask": False},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choices(["quantize", "gather", "experts", "balance", "balance_vjp"],
                       [2, 3, 4, 2, 2])[0]
    if kind == "quantize":
        return {"kind": kind, "experts": _log_int(rng, 1, 128), "rows": rng.randint(1, 768),
                "cols": GROUP * rng.randint(1, 64), "f32": rng.random() < 0.25}
    if kind == "gather":
        cfg = rng.choice(["c2", "c4", "c5", "c6"])
        return {"kind": kind, "cfg": cfg, "proj": rng.choice(["up", "down"]),
                "tokens": _log_int(rng, 1, SHAPES[cfg][4])}
    if kind == "experts":
        cfg = rng.choice(["c2", "c4", "c6"])
        return {"kind": kind, "cfg": cfg, "tokens": _log_int(rng, 1, SHAPES[cfg][4])}
    experts = rng.choice([8, 60, 128, 256, rng.randint(2, 512), 512])
    return {"kind": kind, "tokens": _log_int(rng, 1, 32768), "experts": experts,
            "k": rng.randint(1, min(experts, 10)), "bf16": rng.random() < 0.3,
            "mask": rng.random() < 0.5}


# ------------------------------------------------------------------ inputs
class _Gen:
    """Seeded tensors, one after another."""

    def __init__(self, seed):
        self.dev = torch.device("cuda", torch.cuda.current_device())
        self.g = torch.Generator(device=self.dev)
        self.g.manual_seed(seed * 6007 + 29)

    def normal(self, shape, std=1.0, dtype=torch.float32):
        return (torch.randn(shape, generator=self.g, device=self.dev) * std).to(dtype)


def _encode(w):
    """e2m1 codes (the magnitude's place in E2M1, the sign as bit 3) and scale
    bytes of w [.., cols], groups of 32.  The scale is 2^(floor(log2 max|v|) -
    2); a code is the nearest of the eight magnitudes, ties to the even one."""
    v = w.float().unflatten(-1, (-1, GROUP))
    top = torch.frexp(v.abs().amax(-1)).exponent - 1
    shared = (top - 2).clamp_min(-127)
    a = v.abs() * ((127 - shared) << 23).view(torch.float32)[..., None]
    # the midpoints of neighbours; one between an even and the odd code above it
    # goes down, so there the border is the next value
    mid = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=w.device)
    up = torch.nextafter(mid, mid + 1.0)
    even = torch.arange(7, device=w.device) % 2 == 0
    code = torch.bucketize(a, torch.where(even, up, mid), out_int32=True, right=True)
    return code + 8 * torch.signbit(v), (shared + 127).to(torch.uint8)


def _pack(code):
    """Codes [.., groups, 32] as words [.., groups * 4], the first lowest."""
    c = code.unflatten(-1, (4, 8))
    shift = torch.arange(0, 32, 4, device=code.device, dtype=torch.int32)
    return (c << shift).sum(-1, dtype=torch.int32).flatten(-2)


def _pairs(dev):
    """[256, 2]: the values of a byte's low and high code."""
    v = torch.tensor(E2M1 + [-m for m in E2M1])
    byte = torch.arange(256)
    return torch.stack([v[byte & 15], v[byte >> 4]], 1).to(dev)


def _bank(g, shape):
    """Packed weights [E, N, K / 8] int32 and scales [E, N, K / 32] uint8."""
    E, N, K = shape
    wq = torch.empty((E, N, K // 8), dtype=torch.int32, device=g.dev)
    sc = torch.empty((E, N, K // GROUP), dtype=torch.uint8, device=g.dev)
    for e in range(0, E, 32):
        code, s = _encode(g.normal((min(32, E - e), N, K), 0.02, torch.bfloat16))
        wq[e:e + 32], sc[e:e + 32] = _pack(code), s
    return wq, sc


def _routing(g, tokens, experts, k):
    logits = g.normal((tokens, experts)) + g.normal((experts,), 0.5)
    return logits, logits.topk(k, dim=1).indices.to(torch.int32)


def prepare(case, seed):
    g = _Gen(seed)
    kind = case["kind"]
    if kind == "quantize":
        dtype = torch.float32 if case["f32"] else torch.bfloat16
        shape = (case["experts"], case["rows"], case["cols"])
        return {"case": case, "w": g.normal(shape, 0.02, dtype), "pairs": _pairs(g.dev)}
    if kind in ("balance", "balance_vjp"):
        T, E, K = case["tokens"], case["experts"], case["k"]
        logits, idx = _routing(g, T, E, K)
        st = {"case": case, "logits": logits.bfloat16() if case["bf16"] else logits,
              "idx": idx, "mask": None}
        if case["mask"]:
            # sequences of 256 places, each filled to its own length
            length = 1 + (256 * torch.sigmoid(g.normal(((T + 255) // 256,)) + 1.5)).int()
            pos = torch.arange(T, device=g.dev)
            st["mask"] = pos % 256 < length[pos // 256]
        if kind == "balance_vjp":
            # what the forward pass left, and what comes from above
            keep = st["mask"] if case["mask"] else torch.ones(T, dtype=torch.bool, device=g.dev)
            st["counts"] = _counts(idx, keep, E)
            st["tokens"] = keep.sum(dtype=torch.int32)
            st["dloss"] = torch.full((), 0.01, device=g.dev)
            st["dweights"] = g.normal((T, K), 0.1)
        return st
    d, E, K, f, _ = SHAPES[case["cfg"]]
    if kind == "gather":
        n, k = (f, d) if case["proj"] == "up" else (d, f)
        st = {"case": case, "w": _bank(g, (E, n, k))}
    else:
        k = d
        st = {"case": case, "w": [_bank(g, s) for s in ((E, f, d), (E, f, d), (E, d, f))]}
    st["pairs"] = _pairs(g.dev)
    st["x"] = g.normal((case["tokens"], k), 1.0, torch.bfloat16)
    st["idx"] = _routing(g, case["tokens"], E, K)[1]
    return st


# --------------------------------------------------------------- plain form
def _dequantize(wq, sc, pairs):
    """Weights in f32 of packed words and scales (of normal size, as trained
    weights have); pairs: the two values of each byte of codes."""
    v = pairs[wq.contiguous().view(torch.uint8).int()].flatten(-2)
    scale = (sc.int() << 23).view(torch.float32)
    return (v.unflatten(-1, (-1, GROUP)) * scale[..., None]).flatten(-2)


BLOCK = 64


def _grouped(rows, E):
    """Where the flat rows, sorted by expert, go when every expert's are filled
    up to blocks: (place of each flat row, expert of each block, blocks)."""
    flat = rows.reshape(-1).long()
    n = flat.numel()
    order = torch.argsort(flat, stable=True)
    of = flat[order]
    ones = torch.ones_like(flat)
    counts = torch.zeros(E, dtype=torch.long, device=flat.device).scatter_add_(0, flat, ones)
    blocks = (counts + BLOCK - 1) // BLOCK
    ends = blocks.cumsum(0)
    rank = torch.arange(n, device=flat.device) - (counts.cumsum(0) - counts)[of]
    place = torch.empty_like(flat)
    place[order] = (ends - blocks)[of] * BLOCK + rank
    total = n // BLOCK + min(n, E)
    expert = torch.searchsorted(ends, torch.arange(total, device=flat.device), right=True)
    return place, expert.clamp_max(E - 1), total


def _product(x, bank, route, idx, pairs):
    """x [n, K] (row i for the flat choice i) times its expert's weights."""
    if route is None:  # fewer choices than experts: only those weights
        pick = idx.reshape(-1).long()
        w = _dequantize(bank[0][pick], bank[1][pick], pairs)
        return torch.bmm(w, x[:, :, None])[:, :, 0]
    place, expert, total = route
    xp = torch.zeros((total * BLOCK, x.shape[1]), device=x.device)
    xp[place] = x
    w = _dequantize(*bank, pairs)[expert]
    y = torch.bmm(xp.view(total, BLOCK, -1), w.transpose(1, 2))
    return y.view(total * BLOCK, -1)[place]


def _counts(idx, keep, E):
    c = torch.zeros(E, dtype=torch.int32, device=idx.device)
    take = keep[:, None].expand(idx.shape).reshape(-1).int()
    return c.scatter_add_(0, idx.reshape(-1).long(), take)


def _plain(state):
    case, kind = state["case"], state["case"]["kind"]
    if kind == "quantize":
        w = state["w"]
        code, sc = _encode(w)
        return _dequantize(_pack(code), sc, state["pairs"]).to(w.dtype)
    if kind in ("gather", "experts"):
        x, idx, pairs = state["x"], state["idx"], state["pairs"]
        T, K = idx.shape
        E = SHAPES[case["cfg"]][1]
        route = None if T * K <= E else _grouped(idx, E)
        xf = x.float().repeat_interleave(K, 0)
        if kind == "gather":
            return _product(xf, state["w"], route, idx, pairs).view(T, K, 1, -1).bfloat16()
        gate, up, down = state["w"]
        g = _product(xf, gate, route, idx, pairs)
        h = g / (1.0 + torch.exp(-g)) * _product(xf, up, route, idx, pairs)
        return _product(h, down, route, idx, pairs).view(T, K, -1).bfloat16()
    logits, idx = state["logits"], state["idx"]
    T, E = logits.shape
    K = idx.shape[1]
    z = logits.float()
    p = torch.exp(z - z.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    keep = state["mask"]
    if keep is None:
        keep = torch.ones(T, dtype=torch.bool, device=z.device)
    if kind == "balance":
        counts = _counts(idx, keep, E)
        n = keep.sum(dtype=torch.int32)
        share = 1.0 / n.clamp_min(1).double()
        probs = (p * keep[:, None]).sum(0, dtype=torch.float64) * share
        loss = E * (counts.double() * share / K * probs).sum()
        return {"loss": loss.float(), "counts": counts, "probs": probs.float(), "tokens": n}
    n = state["tokens"].clamp_min(1).float()
    f = state["counts"].float() / (n * K)
    grad = state["dloss"] * E / n * p * (f - (p * f).sum(1, keepdim=True))
    top = z.gather(1, idx.long())
    w = torch.exp(top - top.amax(1, keepdim=True))
    w = w / w.sum(1, keepdim=True)
    dw = state["dweights"]
    grad = grad.scatter_add(1, idx.long(), w * (dw - (w * dw).sum(1, keepdim=True)))
    return (grad * keep[:, None]).to(logits.dtype)


# --------------------------------------------------------- framework's calls
def _ops():
    from __graft_entry__ import load_package

    return load_package()


def _module(state):
    """The expert bank as a program keeps it: views of the same tensors."""
    if "module" not in state:
        nn = _ops().nn
        state["module"] = nn.SplitSwitchFfn(*[
            nn.QuantizedSwitchLinear(wq, sc, None, mode="mxfp4") for wq, sc in state["w"]])
    return state["module"]


def _own(state):
    kind = state["case"]["kind"]
    ops = _ops().ops
    if kind == "quantize":
        wq, sc, _ = ops.quantize(state["w"], mode="mxfp4")
        return ops.dequantize(wq, sc, mode="mxfp4", out_dtype=state["w"].dtype)
    if kind == "gather":
        wq, sc = state["w"]
        return ops.gather_qmm(state["x"][:, None, None, :], wq, sc, rhs_indices=state["idx"],
                              mode="mxfp4")
    if kind == "experts":
        return _module(state).forward(state["x"], state["idx"])
    if kind == "balance":
        loss, counts, probs, tokens = ops.router_balance(state["logits"], state["idx"],
                                                         state["mask"])
        return {"loss": loss, "counts": counts, "probs": probs, "tokens": tokens}
    return ops.router_balance_vjp(state["logits"], state["idx"], state["counts"],
                                  state["tokens"], state["dloss"], state["mask"],
                                  state["dweights"])


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------- work
def work(case):
    kind = case["kind"]
    if kind == "quantize":
        # the weights in and out; codes and scales written and read
        n = case["experts"] * case["rows"] * case["cols"]
        return {"bytes": int(n * (2 * (4 if case["f32"] else 2) + 2 * 4.25 / 8)),
                "flops": 4 * n}
    if kind in ("balance", "balance_vjp"):
        T, E, K = case["tokens"], case["experts"], case["k"]
        es = 2 if case["bf16"] else 4
        b = T * E * es + T * K * 4 + (T if case["mask"] else 0)
        if kind == "balance":
            return {"bytes": b + 8 * E + 8, "flops": 5 * T * E}
        return {"bytes": b + T * E * es + T * K * 4 + 4 * E + 8, "flops": 9 * T * E}
    d, E, K, f, _ = SHAPES[case["cfg"]]
    T = case["tokens"]
    used = E * (1.0 - (1.0 - K / E) ** T)  # experts with a row, uniform routing
    mats = 1 if kind == "gather" else 3
    k, n = (f, d) if case.get("proj") == "down" else (d, f)
    out = n if kind == "gather" else d
    return {"bytes": int(used * mats * d * f * 4.25 / 8 + T * k * 2 + T * K * (4 + 2 * out)),
            "flops": 2 * mats * T * K * d * f}


# -------------------------------------------------------------------- exact
def _pow2(e):
    """2^e in 64 bits, exactly, of a tensor of whole numbers."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _values64(wq, sc):
    table = torch.tensor(E2M1 + [-v for v in E2M1], dtype=torch.float64, device=wq.device)
    parts = [table[((wq >> (4 * i)) & 15).long()] for i in range(8)]
    v = torch.stack(parts, -1).flatten(-2)
    return v * _pow2(sc.long() - 127).repeat_interleave(GROUP, -1)


def _nearest64(w):
    """w with every value replaced by its group's nearest representable one."""
    out = torch.empty(w.shape, dtype=torch.float64, device=w.device)
    for e in range(w.shape[0]):
        v = w[e].double().unflatten(-1, (-1, GROUP))
        big = v.abs().amax(-1, keepdim=True)
        unit = _pow2((torch.floor(torch.log2(big.clamp_min(1e-300))) - 2.0).clamp_min(-127.0))
        a = v.abs() / unit
        step = _pow2(torch.floor(torch.log2(a.clamp_min(1.0))) - 1.0)
        a = (torch.round(a / step) * step).clamp_max(6.0)  # to nearest, ties to even
        out[e] = (torch.copysign(a, v) * unit).flatten(-2)
    return out


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        return _nearest64(st["w"])
    if kind in ("gather", "experts"):
        x, idx = st["x"].double(), st["idx"].long()
        T, K = idx.shape
        banks = [st["w"]] if kind == "gather" else st["w"]
        y = torch.zeros((T, K, banks[-1][0].shape[1]), dtype=torch.float64, device=x.device)
        for e in torch.unique(idx).tolist():
            t, k = (idx == e).nonzero(as_tuple=True)
            w = [_values64(b[0][e], b[1][e]) for b in banks]
            if kind == "gather":
                y[t, k] = x[t] @ w[0].t()
            else:
                g = x[t] @ w[0].t()
                y[t, k] = (g * torch.sigmoid(g) * (x[t] @ w[1].t())) @ w[2].t()
        return y[:, :, None, :] if kind == "gather" else y
    z, idx = st["logits"].double(), st["idx"].long()
    T, E = z.shape
    K = idx.shape[1]
    keep = st["mask"] if st["mask"] is not None else torch.ones(T, device=z.device)
    keep = keep.double()[:, None]
    p = torch.softmax(z, 1)
    chosen = torch.nn.functional.one_hot(idx, E).sum(1).double()
    n = float(keep.sum())
    f = (chosen * keep).sum(0) / max(n * K, 1.0)
    probs = (p * keep).sum(0) / max(n, 1.0)
    if kind == "balance":
        return {"loss": E * (f * probs).sum(), "counts": None, "probs": probs, "tokens": None}
    # d loss / d p = E f / n on kept rows; through the softmax; and the weights'
    up = float(st["dloss"]) * E / max(n, 1.0) * f[None, :].expand(T, E)
    grad = p * (up - (p * up).sum(1, keepdim=True))
    w = torch.softmax(z.gather(1, idx), 1)
    dw = st["dweights"].double()
    inner = w * dw - w * (w * dw).sum(1, keepdim=True)
    grad = grad + torch.zeros_like(z).scatter_add(1, idx, inner)
    return grad * keep
