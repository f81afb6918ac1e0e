"""Cases of the differentiable layer operators (nerf_loam_amd.layers): a matrix product with bias, activation and
residual, 8-bit activation checkpoints, and the embedding lookup with its gradient.

With ``own`` false ``run`` computes each operator in its plain form from elementary torch operations, with ``own`` true
it makes the calls a user makes.  Both take what ``prepare`` returns."""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
MX_BLOCK = 32


def listed():
    return [
        # one sample through one wide layer: the call of a serving loop that answers single queries
        dict(name="linear one row", kind="linear", dtype="bf16", m=1, k=4096, n=4096, act="silu", residual=False),
        # hidden layer of the decoder over the points of a mesh extraction (262144 points at a time)
        dict(name="linear decoder fp32", kind="linear", dtype="fp32", m=262144, k=256, n=256, act="relu", residual=False),
        # a ragged batch: no size is a multiple of a tile or of a vector
        dict(name="linear ragged", kind="linear", dtype="bf16", m=1003, k=1001, n=777, act="gelu", residual=True),
        # training step of a large layer
        dict(name="train wide bf16", kind="train", dtype="bf16", m=16384, k=4096, n=4096, act="gelu", residual=True),
        # training step of a decoder layer in full precision, one scan's samples
        dict(name="train decoder fp32", kind="train", dtype="fp32", m=65536, k=256, n=512, act="silu", residual=False),
        # training step of one tracking batch (2048 rays): small, launches count
        dict(name="train batch fp16", kind="train", dtype="fp16", m=2048, k=256, n=256, act="relu", residual=False),
        # training step whose activations are kept in 8 bits, wide layer
        dict(name="train mx8 wide", kind="train8", dtype="bf16", m=32768, k=2048, n=2048, act="silu", residual=False),
        # the same for a decoder layer over a full scan's samples: long and narrow
        dict(name="train mx8 decoder", kind="train8", dtype="bf16", m=200000, k=256, n=256, act="relu", residual=True),
        # keeping a large activation in 8 bits and getting it back
        dict(name="checkpoint", kind="checkpoint", dtype="bf16", m=131072, k=1024),
        # features of a mapping batch: eight corners of a voxel, weighted; the table of one scan's map
        dict(name="voxel corners", kind="lookup", dtype="bf16", rows=53847, d=16, m=262144, bag=8, scale=1.0, skew=1.0),
        # training step of a token table with a few frequent ids
        dict(name="embedding tokens", kind="embed", dtype="bf16", rows=50000, d=1024, m=32768, bag=1, scale=32.0, skew=3.0),
        # the smallest training step
        dict(name="embedding small", kind="embed", dtype="fp32", rows=1000, d=64, m=512, bag=1, scale=8.0, skew=1.0),
    ]


def _spread(rng, low, high):
    """A whole number whose logarithm is spread evenly, odd ones as likely as even ones"""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "train", "train", "train8", "checkpoint", "lookup", "embed"])
    if kind in ("linear", "train", "train8"):
        dtype = rng.choice(["bf16", "fp16"] if kind == "train8" else ["bf16", "fp16", "fp32"])
        # in full precision a step of relu's derivative next to zero says more about rounding than about the product
        acts = ["none", "gelu", "silu"] if (kind, dtype) == ("train", "fp32") else ["none", "relu", "gelu", "silu"]
        k, n = _spread(rng, 16, 4096), _spread(rng, 1 if kind == "linear" else 8, 4096)
        if rng.random() < 0.5:                            # widths as programs choose them
            k, n = max(16, k // 64 * 64), max(8, n // 64 * 64)
        top = 2.6e11 if dtype == "fp32" else 5.0e11       # M N K of a case: less than the largest listed one
        m = _spread(rng, 1, max(1, min(262144, int(top / 4 / (k * n)), int(2.0e9 / (k + n) / 4))))
        return dict(kind=kind, dtype=dtype, m=m, k=k, n=n, act=rng.choice(acts), residual=rng.random() < 0.5)
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    if kind == "checkpoint":
        k = _spread(rng, 1, 8192)
        return dict(kind=kind, dtype=dtype, m=_spread(rng, 1, max(1, min(262144, 100000000 // k))), k=k)
    d = _spread(rng, 1, 2048)
    bag = rng.choice([1, 1, 2, 8])
    return dict(kind=kind, dtype=dtype, rows=_spread(rng, 1, min(1000000, 100000000 // d)), d=d,
                m=_spread(rng, 1, min(262144, 100000000 // (d * bag))), bag=bag, scale=rng.choice([1.0, 0.5, math.sqrt(d)]), skew=rng.choice([1.0, 3.0]))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dt)

    m = case["m"]
    s = dict(case=case)
    if case["kind"] in ("linear", "train", "train8"):
        k, n = case["k"], case["n"]
        s.update(x=normal(m, k), w=normal(n, k, std=k ** -0.5), b=normal(n, std=0.1), r=normal(m, n) if case["residual"] else None)
        if case["kind"] != "linear":
            s["gy"] = normal(m, n)
            for name in ("x", "w", "b", "r"):
                if s[name] is not None:
                    s[name].requires_grad_(True)
        return s
    if case["kind"] == "checkpoint":
        # rows of very different magnitudes, as behind layers of different depth
        s["x"] = (torch.randn(m, case["k"], generator=g, device="cuda") * torch.exp(torch.randn(m, 1, generator=g, device="cuda"))).to(dt)
        return s
    shape = (m,) if case["bag"] == 1 else (m, case["bag"])
    ids = (torch.rand(shape, generator=g, device="cuda", dtype=torch.float64) ** case["skew"] * case["rows"]).long().clamp_(0, case["rows"] - 1)
    ids = torch.where(torch.rand(shape, generator=g, device="cuda") < 0.01, torch.full_like(ids, -1), ids)      # corners without a row, padding
    s.update(table=normal(case["rows"], case["d"]), ids=ids.to(torch.int32), wt=None)
    if case["bag"] > 1:
        wt = torch.rand(shape, generator=g, device="cuda")
        s["wt"] = wt / wt.sum(1, keepdim=True)
    if case["kind"] == "embed":
        s["gy"] = normal(m, case["d"])
        s["table"].requires_grad_(True)
        if s["wt"] is not None:
            s["wt"].requires_grad_(True)
    return s


# ---- plain forms ----------------------------------------------------------------------------------------------------

def _act(z, act):
    if act == "relu":
        return torch.clamp(z, min=0.0)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "silu":
        s = torch.sigmoid(z)
        return s * (1.0 + z * (1.0 - s))
    return torch.ones_like(z)


def _pow2(e):
    return ((e + 127) << 23).view(torch.float32)


def _mx8(v):
    """The values that 8 bits stand for: blocks of 32 along the last axis share a power of two with which the block's
    largest magnitude is at most 448; below it four significant bits, ties to even, steps of 2^-9 at the small end"""
    rows, cols = v.shape
    b = torch.nn.functional.pad(v.float(), (0, -cols % MX_BLOCK)).view(rows, -1, MX_BLOCK)
    mant, exp = torch.frexp(b.abs().amax(2, keepdim=True))                # amax = mant 2^exp, mant in [1/2, 1)
    e = torch.where(mant > 0.875, exp - 8, exp - 9).clamp(min=-126)       # 448 = 0.875 * 2^9
    q = b * _pow2(-e)
    step = torch.clamp(torch.frexp(q)[1] - 1, min=-6) - 3
    q = torch.round(q * _pow2(-step)) * _pow2(step)
    return (q * _pow2(e)).reshape(rows, -1)[:, :cols]


def _plain_linear(s):
    c, dt = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t() + s["b"].float()
    y = _act(z, c["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    if c["kind"] == "linear":
        return y.to(dt)
    if c["kind"] == "train8":
        x = _mx8(s["x"])
        if c["act"] in ("gelu", "silu"):
            z = _mx8(z)
    dz = s["gy"].float() * _act_slope(z, c["act"])
    out = dict(y=y.to(dt), x=(dz @ w).to(dt), w=(dz.t() @ x).to(dt), b=dz.sum(0).to(dt))
    if s["r"] is not None:
        out["r"] = s["gy"]
    return out


def _plain_embedding(s):
    c, table = s["case"], s["table"]
    ids = s["ids"].long().view(c["m"], c["bag"])
    valid = ids >= 0
    rows = ids.clamp(min=0)
    wt = valid.float() if s["wt"] is None else s["wt"].float() * valid
    y = (table[rows].float() * wt.unsqueeze(2)).sum(1) * c["scale"]
    if c["kind"] == "lookup":
        return y.to(table.dtype)
    # frequent ids make long sums
    g = s["gy"].double() * c["scale"]
    per = (g.unsqueeze(1) * wt.double().unsqueeze(2)).view(-1, c["d"])
    dt = torch.zeros(c["rows"], c["d"], dtype=torch.float64, device="cuda").index_add_(0, rows.view(-1), per)
    out = dict(y=y.to(table.dtype), table=dt.to(table.dtype))
    if s["wt"] is not None:
        out["wt"] = ((g.unsqueeze(1) * table[rows].double()).sum(2) * valid).float()
    return out


def run(state):
    case = state["case"]
    if own:
        return _own(state)
    with torch.no_grad():
        if case["kind"] == "checkpoint":
            return _mx8(state["x"]).to(state["x"].dtype)
        if case["kind"] in ("lookup", "embed"):
            return _plain_embedding(state)
        return _plain_linear(state)


def _own(s):
    from nerf_loam_amd import layers
    c = s["case"]
    if c["kind"] == "checkpoint":
        return layers.checkpoint_decode(layers.checkpoint_encode(s["x"]))
    if c["kind"] == "lookup":
        return layers.embedding_lookup(s["table"], s["ids"], scale=c["scale"], weights=s["wt"])
    if c["kind"] == "embed":
        y = layers.embedding_lookup(s["table"], s["ids"], scale=c["scale"], weights=s["wt"])
        names = ["table"] + (["wt"] if s["wt"] is not None else [])
    else:
        y = layers.linear_act(s["x"], s["w"], s["b"], act=c["act"], residual=s["r"], checkpoint="mx8" if c["kind"] == "train8" else None)
        if c["kind"] == "linear":
            return y
        names = ["x", "w", "b"] + (["r"] if s["r"] is not None else [])
    grads = torch.autograd.grad(y, [s[n] for n in names], s["gy"])
    return dict(y=y.detach(), **dict(zip(names, grads)))


# ---- the definition in 64 bits --------------------------------------------------------------------------------------

def _exact_codes(v):
    """values of the 8-bit format by search: the nearest of all 127 magnitudes, the even code on a tie"""
    mags = torch.tensor([(c % 8) * 2.0 ** -9 if c < 8 else (1 + (c % 8) / 8) * 2.0 ** (c // 8 - 7) for c in range(127)], dtype=torch.float64, device=v.device)
    rows, cols = v.shape
    nb = -(-cols // MX_BLOCK)
    pad = torch.zeros(rows, nb * MX_BLOCK, dtype=torch.float64, device=v.device)
    pad[:, :cols] = v
    blocks = pad.view(-1, MX_BLOCK)
    out = torch.empty_like(blocks)
    for i in range(0, len(blocks), 1 << 20):
        b = blocks[i:i + (1 << 20)]
        top = b.abs().max(1, keepdim=True).values
        e = torch.ceil(torch.log2(torch.clamp(top, min=2.0 ** -300) / 448.0)).clamp(min=-126)
        e = torch.where(top > 448.0 * torch.exp2(e), e + 1, torch.where((top <= 224.0 * torch.exp2(e)) & (e > -126), e - 1, e))
        a = b.abs() * torch.exp2(-e)
        hi = torch.searchsorted(mags, a).clamp(max=126)
        lo = (hi - 1).clamp(min=0)
        up, down = mags[hi] - a, a - mags[lo]
        code = torch.where(up < down, hi, torch.where(up > down, lo, torch.where(hi % 2 == 0, hi, lo)))
        out[i:i + (1 << 20)] = torch.copysign(mags[code], b) * torch.exp2(e)
    return out.view(rows, -1)[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    f = torch.nn.functional
    curve = {"none": lambda t: t, "relu": f.relu, "gelu": f.gelu, "silu": f.silu}
    if case["kind"] == "checkpoint":
        return _exact_codes(s["x"].double())
    if case["kind"] in ("lookup", "embed"):
        table = s["table"].detach().double()
        table = torch.cat([table, torch.zeros_like(table[:1])]).requires_grad_(True)         # the last row stands for no row
        ids = torch.where(s["ids"] < 0, torch.full_like(s["ids"], case["rows"]), s["ids"]).long()
        wt = None if s["wt"] is None else s["wt"].detach().double().requires_grad_(True)
        picked = f.embedding(ids, table)
        y = case["scale"] * (picked if wt is None else torch.matmul(wt.unsqueeze(1), picked).squeeze(1))
        if case["kind"] == "lookup":
            return y.detach()
        grads = torch.autograd.grad(y, [table] + ([wt] if wt is not None else []), s["gy"].double())
        out = dict(y=y.detach(), table=grads[0][:-1])
        if wt is not None:
            out["wt"] = grads[1]
        return out
    x, w, b = (s[n].detach().double() for n in ("x", "w", "b"))
    z = f.linear(x, w, b).requires_grad_(True)
    a = curve[case["act"]](z)
    y = (a if s["r"] is None else a + s["r"].detach().double()).detach()
    if case["kind"] == "linear":
        return y
    if case["kind"] == "train8":
        x = _exact_codes(x)
        if case["act"] in ("gelu", "silu"):
            z = _exact_codes(z.detach()).requires_grad_(True)
            a = curve[case["act"]](z)
    dz, = torch.autograd.grad(a, z, s["gy"].double())
    out = dict(y=y, x=torch.mm(dz, w), w=torch.mm(dz.t(), x), b=dz.sum(0))
    if s["r"] is not None:
        out["r"] = None
    return out


def work(case):
    """Each input read once and each output written once; multiplications and additions of the products"""
    es = 4 if case["dtype"] == "fp32" else 2
    m = case["m"]
    if case["kind"] in ("linear", "train", "train8"):
        k, n = case["k"], case["n"]
        r = m * n if case["residual"] else 0
        forward = m * k + n * k + n + m * n + r
        if case["kind"] == "linear":
            return {"bytes": forward * es, "flops": 2 * m * n * k}
        return {"bytes": (forward + m * n + m * k + n * k + n) * es, "flops": 6 * m * n * k}
    if case["kind"] == "checkpoint":
        return {"bytes": 2 * m * case["k"] * es, "flops": 0}
    look = m * case["bag"]
    touched = min(look, case["rows"]) * case["d"] * es          # a row asked for twice is read once
    weights = 4 * look if case["bag"] > 1 else 0
    out = m * case["d"] * es
    if case["kind"] == "lookup":
        return {"bytes": touched + 4 * look + weights + out, "flops": 2 * look * case["d"]}
    return {"bytes": touched + 4 * look + 2 * weights + 2 * out + case["rows"] * case["d"] * es, "flops": 6 * look * case["d"]}
