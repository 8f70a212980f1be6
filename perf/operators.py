"""Cases that measure the 8-bit optimizer step and the head's loss against their plain forms.

Two families:

  "adam"  one AdamW step over all tensors of a model with the moments in 8 bits (m: E4M3, v: an
          unsigned float of five exponent and three fraction bits, one power-of-two scale per 256
          places of the flat, rounding dithered by a hash of place and step), clip by the global
          norm, decay of matrices, bf16 twins; afterwards the moments are read as bf16 values.
  "loss"  softmax cross entropy of the language model's head, logits = x W + b over the whole
          vocabulary, per token; with grad set also dx, and dW and db added to the gradient flat.

`run` computes them with elementary torch operations while `own` is false and calls the framework
while it is true.  `exact` states the definitions again in 64 bits, by other means.
"""
import math

import torch

own = False

BLOCK = 256          # places of the flat that share a scale
GOLD, MULT, M32 = 0x9E3779B9, 0xB7E15163, 0xFFFFFFFF
HYPER = {"beta1": 0.9, "beta2": 0.95, "eps": 1e-8, "weight_decay": 0.1, "grad_clip": 1.0}
LR, GRAD_SCALE = 3e-4, 1.0
ADAM_MOST = 168_000_000                 # elements of the largest drawn optimizer flat
LOSS_MOST = 4096 * 1536 * 100_000       # rows * d * vocab of the largest drawn loss


# ---- cases ---------------------------------------------------------------------------------

def _adam(name, d, ff, blocks, vocab, grad, t, clipped):
    return {"name": name, "op": "adam", "d": d, "ff": ff, "blocks": blocks, "vocab": vocab, "grad": grad,
            "t": t, "clipped": clipped}


def _loss(name, rows, d, vocab, grad, out, pad, bias):
    return {"name": name, "op": "loss", "rows": rows, "d": d, "vocab": vocab, "grad": grad, "out": out,
            "pad": pad, "bias": bias}


def listed():
    return [
        # the test model's 26 tensors: the call's latency
        _adam("adam tiny f32", 64, 256, 2, 256, "f32", 1, False),
        # nothing divides anything: tensors begin and end inside blocks and tiles; E4M3 gradients with scales
        _adam("adam ragged fp8", 333, 1001, 3, 10007, "fp8", 12345, True),
        # the 185M model, float gradients as its training run has them, and bf16 ones
        _adam("adam 185m f32", 1024, 4096, 12, 16384, "f32", 100, True),
        _adam("adam 185m bf16", 1024, 4096, 12, 16384, "bf16", 2000, False),
        # one token scored while a model is compared or sampled from: latency, the weights are read once
        _loss("loss 185m one token", 1, 1024, 16384, False, "f32", 0.0, True),
        # a held-out text at an odd vocabulary, rows that are not 16-byte aligned
        _loss("loss ragged", 517, 712, 50257, False, "f32", 0.3, False),
        # one context of the 555M model evaluated
        _loss("loss 555m 2048 tokens", 2048, 1536, 100000, False, "f32", 0.0, True),
        # the test model's training step
        _loss("grad tiny f32", 254, 64, 256, True, "f32", 0.0, True),
        # packed short documents, over half of the rows are padding, odd everything
        _loss("grad ragged f32", 777, 331, 10007, True, "f32", 0.55, True),
        # a 4096-token microbatch of the 185M model into a float gradient flat
        _loss("grad 185m f32", 4096, 1024, 16384, True, "f32", 0.0, True),
        # a short fine-tuning batch of the 555M model: few rows, large vocabulary, bf16 gradients
        _loss("grad 555m 96 tokens bf16", 96, 1536, 100000, True, "bf16", 0.1, True),
        # a 4096-token microbatch of the 555M model into a bf16 gradient flat
        _loss("grad 555m bf16", 4096, 1536, 100000, True, "bf16", 0.0, True),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    if rng.random() < 0.4:
        while True:
            d = _spread(rng, 48, 1100)
            c = _adam("", d, _spread(rng, 2 * d, 5 * d), rng.randint(1, 12), _spread(rng, 200, 60000),
                      rng.choice(["f32", "bf16", "fp8"]), _spread(rng, 1, 100000), rng.random() < 0.5)
            if sum(n for n, _ in tensors_of(c)) <= ADAM_MOST:
                break
    else:
        while True:
            c = _loss("", _spread(rng, 1, 8192), _spread(rng, 33, 2048), _spread(rng, 130, 100000),
                      rng.random() < 0.65, rng.choice(["f32", "bf16"]), rng.choice([0.0, 0.0, 0.2, 0.7]),
                      rng.random() < 0.7)
            if rng.random() < 0.5:      # sizes as models have them, beside whatever the spread gives
                c["d"], c["vocab"] = (c["d"] + 63) // 64 * 64, (c["vocab"] + 127) // 128 * 128
            if c["rows"] * c["d"] * c["vocab"] * (2 if c["out"] == "f32" else 1) <= LOSS_MOST:
                break
    del c["name"]
    return c


def tensors_of(case):
    """(elements, is a matrix) of the model's tensors in registration order."""
    d, ff = case["d"], case["ff"]
    block = [(3 * d * d, True), (3 * d, False), (d * d, True), (d, False), (d * ff, True), (ff, False),
             (ff * d, True), (d, False), (d, False), (d, False), (d, False), (d, False)]
    return [(d * case["vocab"], True), (case["vocab"], False)] + block * case["blocks"]


# ---- 8-bit moments: the plain form -----------------------------------------------------------

def _pow2(e):
    """2^e as float64, exactly, for a tensor of whole numbers."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _whole_blocks(x, n_blocks):
    out = torch.zeros(n_blocks * BLOCK, dtype=x.dtype, device=x.device)
    out[: x.numel()] = x
    return out.view(n_blocks, BLOCK)


def _scales(x, n_blocks):
    """The exponent byte of each block of a float32 flat: the least exponent at which 1.75 * 2^E covers it."""
    u = _whole_blocks(x.abs().view(torch.int32), n_blocks).amax(1).to(torch.int64)
    return ((u + 0x1FFFFF) >> 23).clamp(max=255)


def _spread_exponents(byte, n):
    return (byte.clamp(min=1) - 127).repeat_interleave(BLOCK)[:n]


def _quantise(x, byte, normals, dither):
    """Values of a non-negative float32 flat on its grid: `normals` binades with eight steps each, then even steps down to 0."""
    n = x.numel()
    x = x.double()
    top = _spread_exponents(byte, n)
    e = torch.frexp(x)[1].to(torch.int64) - 1
    step = torch.maximum(e, top - (normals - 1)) - 3
    k = torch.round(x * _pow2(20 - step)) + dither.double()
    return torch.floor(k * 2.0 ** -20), step


def _hash(n, t, device):
    i = torch.arange(n, dtype=torch.int64, device=device)
    s = ((t * GOLD) & M32) ^ (t & M32) >> 7
    s = (s * MULT) & M32
    x = (i * GOLD + (s ^ s >> 16)) & M32
    x ^= x >> 15
    x = (x * MULT) & M32
    return x ^ x >> 15


def _plain_adam(s):
    c, n, h = s["case"], s["n"], HYPER
    s["t"] += 1
    t, nb = s["t"], s["n_blocks"]
    g = s["g"]
    if c["grad"] == "fp8":
        g = g.view(torch.float8_e4m3fn).float() * s["gscale"][s["seg"]]
    x = g.double() * GRAD_SCALE
    norm = torch.sqrt((x * x).sum())
    gs = torch.where(norm > h["grad_clip"], GRAD_SCALE * (h["grad_clip"] / (norm + 1e-12)),
                     torch.full_like(norm, GRAD_SCALE))
    x = g.double() * gs
    del g
    # the moments as they are stored: E4M3 codes and codes of the unsigned format, times their block's scale
    em = _spread_exponents(s["m_exp"].to(torch.int64), n)
    m = (s["m"][:n].view(torch.float8_e4m3fn).double() * _pow2(em - 8)).float()
    code = s["v"][:n].to(torch.int64)
    field = code >> 3
    frac = (code & 7).double() + torch.where(field > 0, 8.0, 0.0)
    ev = _spread_exponents(s["v_exp"].to(torch.int64), n)
    v = (frac * _pow2(field.clamp(min=1) - 34 + ev)).float()
    del em, ev, code, field, frac
    m = (h["beta1"] * m.double() + (1.0 - h["beta1"]) * x).float()
    v = (h["beta2"] * v.double() + ((1.0 - h["beta2"]) * x) * x).float()
    del x
    mhat = m.double() / (1.0 - h["beta1"] ** t)
    vhat = v.double() / (1.0 - h["beta2"] ** t)
    p = (s["p"].double() - (LR * mhat) / (torch.sqrt(vhat) + h["eps"])).float()
    del mhat, vhat
    p = torch.where(s["matrix"], (p.double() - (LR * h["weight_decay"]) * p.double()).float(), p)
    s["p"].copy_(p)
    s["twin"].copy_(torch.where(s["matrix"], p.bfloat16(), s["twin"]))
    s["g"].zero_()
    del p
    z = _hash(n, t, m.device)
    bm = _scales(m, nb)
    q, step = _quantise(m.abs(), bm, 15, (z & 0xFFFF) << 4)
    value = q * _pow2(step)
    s["m_out"].copy_(torch.copysign(value, m.double()).float())
    top = _spread_exponents(bm, n)
    code = (value * _pow2(8 - top)).float().to(torch.float8_e4m3fn).view(torch.uint8)
    s["m"][:n] = code | torch.where(torch.signbit(m), 128, 0).to(torch.uint8)
    s["m_exp"].copy_(bm)
    bv = _scales(v, nb)
    q, step = _quantise(v, bv, 31, (z >> 16) << 4)
    q = torch.where(v > 0, q.clamp(min=1.0), q)
    value = q * _pow2(step)
    s["v_out"].copy_(value.float())
    top = _spread_exponents(bv, n)
    q = q.to(torch.int64)
    field = step + 3 - top + 31                         # of the binade the step belongs to
    field = torch.where(q >= 8, field, torch.zeros_like(field))
    field, q = field + (q >> 4), torch.where(q >= 16, q >> 1, q)
    s["v"][:n] = ((field << 3) + torch.where(q >= 8, q - 8, q)).to(torch.uint8)
    s["v_exp"].copy_(bv)
    return {"p": s["p"], "twin": s["twin"], "g": s["g"], "m": s["m_out"], "v": s["v_out"]}


# ---- the head's loss: the plain form -----------------------------------------------------------

def _plain_loss(s):
    c = s["case"]
    x, target = s["x"].float(), s["target"].long()
    live = (target >= 0) & (target < c["vocab"])
    w = s["w"].float()
    logits = x @ w
    if c["bias"]:
        logits = logits + s["b"]
    top = logits.max(1, keepdim=True).values
    lse = top + torch.log(torch.exp(logits - top).sum(1, keepdim=True))
    at = torch.where(live, target, torch.zeros_like(target)).unsqueeze(1)
    nll = torch.where(live, (lse - logits.gather(1, at)).squeeze(1), torch.zeros_like(lse.squeeze(1)))
    if not c["grad"]:
        return {"nll": nll}
    delta = torch.exp(logits - lse)
    delta.scatter_add_(1, at, torch.full_like(lse, -1.0))
    delta *= torch.where(live, s["scale"], 0.0).float().unsqueeze(1)
    s["dx"].copy_(delta @ w.t())
    s["dw"].copy_(s["dw"].float() + x.t() @ delta)
    s["db"].copy_(s["db"].float() + delta.sum(0))
    return {"nll": nll, "dx": s["dx"], "dw": s["dw"], "db": s["db"]}


# ---- inputs ------------------------------------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _prepare_adam(case, seed):
    gen = _generator(seed)
    rows = tensors_of(case)
    sizes = torch.tensor([n for n, _ in rows], device="cuda")
    n = int(sum(k for k, _ in rows))
    nb = (n + BLOCK - 1) // BLOCK

    def normal(std):
        return torch.empty(n, device="cuda").normal_(0.0, std, generator=gen)

    s = {"case": case, "n": n, "n_blocks": nb, "t": case["t"] - 1, "rows": rows}
    s["matrix"] = torch.tensor([x for _, x in rows], device="cuda").repeat_interleave(sizes)
    # the tensors' gradients differ in size: a factor of up to a few hundred between them
    size = torch.empty(len(rows), device="cuda").uniform_(-3.0, 3.0, generator=gen).exp_()
    unit = size.repeat_interleave(sizes)
    unit *= (2.5 if case["clipped"] else 0.4) / float(unit.double().square().sum().sqrt())
    s["p"] = normal(0.02)
    grad = normal(1.0) * unit
    if case["grad"] == "fp8":
        s["seg"] = torch.arange(len(rows), dtype=torch.int32, device="cuda").repeat_interleave(sizes)
        s["gscale"] = torch.zeros(len(rows), device="cuda").scatter_reduce_(
            0, s["seg"].long(), grad.abs(), "amax") / 448.0
        s["g"] = (grad / s["gscale"][s["seg"]]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        s["g"] = grad if case["grad"] == "f32" else grad.bfloat16()
    # the state in the middle of a run (the first step finds zeros): codes and exponents as they are stored
    s["m"] = torch.zeros(nb * BLOCK, dtype=torch.uint8, device="cuda")
    s["v"] = torch.zeros(nb * BLOCK, dtype=torch.uint8, device="cuda")
    s["m_exp"] = torch.zeros(nb, dtype=torch.uint8, device="cuda")
    s["v_exp"] = torch.zeros(nb, dtype=torch.uint8, device="cuda")
    if case["t"] > 1:
        m = normal(0.3) * unit
        v = (normal(1.0) * unit) ** 2 + (0.1 * unit) ** 2
        bm, bv = _scales(m, nb), _scales(v, nb)
        tm, tv = _spread_exponents(bm, n), _spread_exponents(bv, n)
        s["m"][:n] = (m.double() * _pow2(8 - tm)).float().to(torch.float8_e4m3fn).view(torch.uint8)
        e = torch.maximum(torch.frexp(v.double())[1].to(torch.int64) - 1, tv - 30)
        s["v"][:n] = (((e - tv + 31) << 3) + torch.floor(v.double() * _pow2(3 - e)).to(torch.int64) - 8).to(torch.uint8)
        s["m_exp"].copy_(bm)
        s["v_exp"].copy_(bv)
    s["twin"] = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    s["m_out"] = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    s["v_out"] = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    if own:
        s = _into_arena(s)
    return s


class _At:
    """Device memory of the library's for torch.as_tensor."""

    def __init__(self, keep, ptr, n, kind):
        self.keep = keep
        self.__cuda_array_interface__ = {"shape": (n,), "typestr": kind, "data": (ptr, False), "version": 3}


def _into_arena(s):
    """The handle a training program keeps, holding the same state."""
    from anni_amd import lib
    from anni_amd.lm_adam import LmAdam

    case, n, nb = s["case"], s["n"], s["n_blocks"]
    kinds = {"f32": (lib.F32, "<f4"), "bf16": (lib.BF16, "<i2"), "fp8": (lib.FP8_E4M3, "|u1")}
    flags = lib.T_DECAY | lib.T_TWIN
    opt = LmAdam([(k, flags if matrix else 0) for k, matrix in s["rows"]], grad_type=kinds[case["grad"]][0],
                 moment_type=lib.Q8, twins=True, skip_nonfinite=True, **HYPER)
    o = opt.o
    o.t = s["t"]

    def view(ptr, k, kind, dtype):
        return torch.as_tensor(_At(opt, ptr, k, kind), device="cuda").view(dtype)

    dtype = s["g"].dtype
    out = {"case": case, "opt": opt, "m_out": s["m_out"], "v_out": s["v_out"],
           "p": view(o.d_param, n, "<f4", torch.float32), "g": view(o.d_grad, n, kinds[case["grad"]][1], dtype),
           "twin": view(o.d_param_bf16, n, "<i2", torch.bfloat16)}
    out["p"].copy_(s["p"])
    out["g"].copy_(s["g"])
    view(o.d_m, nb * BLOCK, "|u1", torch.uint8).copy_(s["m"])
    view(o.d_v, nb * BLOCK, "|u1", torch.uint8).copy_(s["v"])
    view(o.d_m + nb * BLOCK, nb, "|u1", torch.uint8).copy_(s["m_exp"])
    view(o.d_v + nb * BLOCK, nb, "|u1", torch.uint8).copy_(s["v_exp"])
    if case["grad"] == "fp8":
        view(o.d_gscale, len(s["rows"]), "<f4", torch.float32).copy_(s["gscale"])
    torch.cuda.synchronize()
    return out


def _prepare_loss(case, seed):
    gen = _generator(seed)
    rows, d, vocab = case["rows"], case["d"], case["vocab"]
    kind = torch.float32 if case["out"] == "f32" else torch.bfloat16

    def normal(*shape, std=1.0):
        return torch.empty(*shape, device="cuda").normal_(0.0, std, generator=gen)

    s = {"case": case, "x": normal(rows, d).bfloat16(), "w": normal(d, vocab, std=2.0 / math.sqrt(d)).bfloat16(),
         "b": normal(vocab, std=0.5)}
    # frequent tokens are frequent; rows without a target are padding
    u = torch.empty(rows, device="cuda").uniform_(0.0, 1.0, generator=gen)
    s["target"] = (torch.exp(u * math.log(vocab + 1.0)) - 1.0).long().clamp(0, vocab - 1).int()
    pad = torch.empty(rows, device="cuda").uniform_(0.0, 1.0, generator=gen) < case["pad"]
    s["target"][pad] = -1
    s["nll"] = torch.zeros(rows, device="cuda")
    s["scale"] = 1.0 / max(1, rows)
    if case["grad"]:
        s["dx"] = torch.zeros(rows, d, dtype=kind, device="cuda")
        # what earlier microbatches left in the gradient flat
        s["dw"] = normal(d, vocab, std=1e-3 / math.sqrt(rows)).to(kind)
        s["db"] = normal(vocab, std=1e-3 / math.sqrt(rows)).to(kind)
    if own:
        from anni_amd import lib
        from anni_amd.head_loss import HeadLoss

        s["plan"] = HeadLoss(rows, d, vocab, grad_type=lib.F32 if case["out"] == "f32" else lib.BF16,
                             grad=case["grad"])
        torch.cuda.synchronize()
    return s


def prepare(case, seed):
    return _prepare_adam(case, seed) if case["op"] == "adam" else _prepare_loss(case, seed)


def run(state):
    case = state["case"]
    if not own:
        return _plain_adam(state) if case["op"] == "adam" else _plain_loss(state)
    s = state
    if case["op"] == "adam":
        s["opt"].step_scaled(LR, GRAD_SCALE)
        s["opt"].read_moments(s["m_out"].data_ptr(), s["v_out"].data_ptr())
        return {"p": s["p"], "twin": s["twin"], "g": s["g"], "m": s["m_out"], "v": s["v_out"]}
    bias = s["b"].data_ptr() if case["bias"] else None
    if not case["grad"]:
        s["plan"].run(s["x"].data_ptr(), s["w"].data_ptr(), bias, s["target"].data_ptr(), s["nll"].data_ptr())
        return {"nll": s["nll"]}
    s["plan"].run(s["x"].data_ptr(), s["w"].data_ptr(), bias, s["target"].data_ptr(), s["nll"].data_ptr(),
                  scale=s["scale"], dx=s["dx"].data_ptr(), dw=s["dw"].data_ptr(), db=s["db"].data_ptr())
    return {"nll": s["nll"], "dx": s["dx"], "dw": s["dw"], "db": s["db"]}


def work(case):
    if case["op"] == "adam":
        n = sum(k for k, _ in tensors_of(case))
        mats = sum(k for k, x in tensors_of(case) if x)
        g = {"f32": 4, "bf16": 2, "fp8": 1}[case["grad"]]
        # p, g and both moments read and written, twins and the moments' bf16 values written; about 20 operations each
        return {"bytes": n * (8 + 2 * g + 4 + 4) + 2 * mats + 4 * (n // BLOCK), "flops": 20 * n}
    rows, d, vocab = case["rows"], case["d"], case["vocab"]
    out = 4 if case["out"] == "f32" else 2
    nbytes = 2 * rows * d + 2 * d * vocab + 4 * vocab + 8 * rows
    if not case["grad"]:
        return {"bytes": nbytes, "flops": 2 * rows * d * vocab}
    return {"bytes": nbytes + out * (rows * d + 2 * d * vocab + 2 * vocab), "flops": 6 * rows * d * vocab}


# ---- the definitions in 64 bits ----------------------------------------------------------------

def _grid(normals):
    """All magnitudes of a format with eight steps to the binade, `normals` binades, the top one at 1..1.75 (1.875 left out)."""
    sub = [k * 2.0 ** (-(normals - 1) - 3) for k in range(8)]
    nor = [(1 + k / 8) * 2.0 ** (e - (normals - 1)) for e in range(normals) for k in range(8)]
    return torch.tensor((sub + nor)[:-1], dtype=torch.float64, device="cuda")


def _exact_store(x, t, high, grid, floor):
    """Where the stored values of a non-negative float flat lie: between two neighbours of the grid the dither decides."""
    n = x.numel()
    nb = (n + BLOCK - 1) // BLOCK
    full = torch.zeros(nb * BLOCK, dtype=torch.float64, device=x.device)
    full[:n] = x
    full = full.view(nb, BLOCK)
    top = full.amax(1, keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=2.0 ** -126)))
    scale = torch.exp2(e)
    scale = torch.where(scale > top.clamp(min=2.0 ** -126), scale / 2, scale)
    scale = torch.where(2 * scale <= top, scale * 2, scale)
    scale = torch.where(top > 1.75 * scale, scale * 2, scale)
    y = (full / scale).view(-1)[:n]
    lo = torch.searchsorted(grid, y, right=True) - 1
    hi = (lo + 1).clamp(max=grid.numel() - 1)
    gap = torch.where(hi > lo, grid[hi] - grid[lo], torch.ones_like(y))
    place = torch.round((y - grid[lo]) / gap * 1048576.0)        # of 2^20 between the neighbours
    s = (t * GOLD % 2 ** 32) ^ (t >> 7)
    s = s * MULT % 2 ** 32
    s ^= s >> 16
    i = torch.arange(n, device=x.device)
    z = torch.remainder(i * GOLD + s, 2 ** 32)
    z = torch.bitwise_xor(z, z // 2 ** 15)
    z = torch.remainder(((z >> 16) * MULT % 2 ** 16 << 16) + (z & 0xFFFF) * MULT, 2 ** 32)
    z = torch.bitwise_xor(z, z // 2 ** 15)
    z = z // 2 ** 16 if high else z % 2 ** 16
    at = torch.where(place + 16.0 * z >= 1048576.0, hi, lo)
    if floor:
        at = torch.where((y > 0) & (at == 0), torch.ones_like(at), at)
    return grid[at] * scale.expand(nb, BLOCK).reshape(-1)[:n]


def _exact_adam(case, seed):
    global own
    kept, own = own, False
    try:
        s = _prepare_adam(case, seed)
    finally:
        own = kept
    n, t = s["n"], case["t"]
    rows = s["rows"]
    ends = torch.tensor([k for k, _ in rows], device="cuda").cumsum(0)
    e4m3, e5m3 = _grid(15), _grid(31)
    byte = s["m"][:n].long()
    blk = torch.arange(n, device="cuda") // BLOCK
    m = e4m3[(byte & 127)] * torch.where(byte > 127, -1.0, 1.0) * torch.exp2(s["m_exp"].double().clamp(min=1) - 127)[blk]
    v = e5m3[s["v"][:n].long()] * torch.exp2(s["v_exp"].double().clamp(min=1) - 127)[blk]
    m, v = m.float().double(), v.float().double()
    if case["grad"] == "fp8":
        sign = torch.where(s["g"] > 127, -1.0, 1.0).double()
        which = torch.bucketize(torch.arange(n, device="cuda"), ends, right=True)
        g = (e4m3[(s["g"].long() & 127)] * 256.0 * sign).float() * s["gscale"][which]
    else:
        g = s["g"]
    g = g.double()
    norm = float((g * g).sum().sqrt())
    g = g * (1.0 / (norm + 1e-12) if norm > 1.0 else 1.0)
    m = (0.9 * m + (1 - 0.9) * g).float().double()
    v = (0.95 * v + (1 - 0.95) * g * g).float().double()
    p = s["p"].double() - 3e-4 * (m / (1 - 0.9 ** t)) / ((v / (1 - 0.95 ** t)).sqrt() + 1e-8)
    matrix = torch.tensor([x for _, x in rows], device="cuda")[
        torch.bucketize(torch.arange(n, device="cuda"), ends, right=True)]
    p = torch.where(matrix, p * (1 - 3e-4 * 0.1), p)
    return {"p": p, "twin": torch.where(matrix, p, torch.zeros_like(p)), "g": None,
            "m": torch.copysign(_exact_store(m.abs(), t, False, e4m3, False), m),
            "v": _exact_store(v, t, True, e5m3, True)}


def _exact_loss(case, seed):
    global own
    kept, own = own, False
    try:
        s = _prepare_loss(case, seed)
    finally:
        own = kept
    rows, vocab = case["rows"], case["vocab"]
    x, w = s["x"].double(), s["w"].double()
    z = torch.mm(x, w)
    if case["bias"]:
        z += s["b"].double()
    lse = torch.logsumexp(z, 1)
    use = s["target"] >= 0
    r = torch.arange(rows, device="cuda")[use]
    k = s["target"][use].long()
    nll = torch.zeros(rows, dtype=torch.float64, device="cuda")
    nll[r] = lse[r] - z[r, k]
    if not case["grad"]:
        return {"nll": nll}
    z.sub_(lse.unsqueeze(1)).exp_()
    z[r, k] -= 1.0
    z[~use] = 0.0
    z *= s["scale"]
    return {"nll": nll, "dx": torch.mm(z, w.t()), "dw": s["dw"].double() + torch.mm(x.t(), z),
            "db": s["db"].double() + z.sum(0)}


def exact(case, seed):
    return _exact_adam(case, seed) if case["op"] == "adam" else _exact_loss(case, seed)
