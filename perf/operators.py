"""Cases of the pair-stream operators: what makes, updates and reads the pair representation ``(B, N_i, N_j, D)``
around the triangle update.

Operators (``op``):

* ``dropout``  -- ``residual + dropout(update)``; the mask comes from a counter-based generator and is never stored.
* ``norm``     -- the same addition, and the root-mean-square norm of its result.
* ``norm_fp8`` -- the same, with the norm's output in e4m3 and fp32 scales.
* ``embed``    -- embedding lookup with scaling, added to a base, and its gradient.

``run`` computes them in elementary torch operations, or, where ``own`` is true, through the framework.
``grad`` says whether the pass is a training step (forward and gradients) or the forward alone.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
_EPS = 1e-5
_E4M3_MAX = 448.0


def _pair(name, op, b, i, j, d, dtype, grad, p=0.0, shared="none", residual=True, layout="whole", group=0):
    case = dict(op=op, b=b, i=i, j=j, d=d, dtype=dtype, grad=grad, p=p, shared=shared, residual=residual, layout=layout)
    if op == "norm_fp8":
        case["group"] = group
    return dict(name=name, **case) if name else case


def _embed(name, b, i, j, d, dtype, grad, v, index, bins, base, scale):
    case = dict(op="embed", b=b, i=i, j=j, d=d, dtype=dtype, grad=grad, v=v, index=index, bins=bins, base=base, scale=scale)
    return dict(name=name, **case) if name else case


def listed():
    return [
        # one token's row through the norm, as a head that reads a single position does: latency
        _pair("norm_one_row", "norm", 1, 1, 1, 512, "bf16", False),
        # a training crop of 384 residues at the width of the pair stack, dropout shared over rows: the update's way
        # back into the stream and the next block's norm, forward and backward
        _pair("norm_train_crop384", "norm", 1, 384, 384, 128, "bf16", True, p=0.25, shared="rows"),
        # fp32 training without dropout on a batch of two
        _pair("norm_train_fp32", "norm", 2, 256, 256, 256, "fp32", True),
        # an odd token count, a width that no vector load divides, no residual
        _pair("norm_odd_width", "norm", 2, 203, 197, 131, "fp16", False, residual=False),
        # serving: N = 1024, D = 256, the norm's output quantised for an 8-bit product
        _pair("norm_fp8_1024", "norm_fp8", 1, 1024, 1024, 256, "bf16", False, group=128),
        # the block of one rank of a row-sharded grid, scale per row, wide rows
        _pair("norm_fp8_block", "norm_fp8", 1, 96, 768, 384, "bf16", False, layout="block", group=0),
        # sampling with dropout left on, every element its own: N = 1024, D = 256
        _pair("dropout_1024", "dropout", 1, 1024, 1024, 256, "bf16", False, p=0.25),
        # a small training crop, mask shared over columns, both inputs transposed views (the incoming update's view)
        _pair("dropout_train_small", "dropout", 1, 72, 72, 128, "bf16", True, p=0.25, shared="columns", layout="transposed"),
        # relative-position bins into the stream: 2 x 32 + 2 rows, N = 1024
        _embed("embed_relpos_1024", 1, 1024, 1024, 256, "bf16", False, 66, "int32", "relpos", True, 1.0),
        # the same in training, on a crop of 768 with padded positions (index -1)
        _embed("embed_relpos_train", 1, 768, 768, 128, "bf16", True, 66, "int64", "padded", True, 1.0),
        # residue types: a short sequence in fp32, latency
        _embed("embed_tokens_train", 2, 1, 500, 384, "fp32", True, 21, "int64", "uniform", False, math.sqrt(384.0)),
        # a large vocabulary with skewed frequencies
        _embed("embed_vocab_train", 4, 1, 8192, 512, "bf16", True, 32000, "int64", "skewed", False, 1.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_fp8", "dropout", "embed", "embed"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    grad = op != "norm_fp8" and rng.random() < 0.6
    d = rng.choice([64, 128, 128, 256, 384, 512, _log(rng, 32, 1024), _log(rng, 1024, 4096)])
    # elements of one tensor: from a row to what the largest listed passes move
    most = ((1 << 26) if grad else (1 << 28)) // _BYTES[dtype]
    rows = max(1, min(_log(rng, 1, 1 << 20), most // d))
    b = rng.choice([1, 1, 2, 3]) if rows >= 8 else 1
    i = max(1, int(round(math.sqrt(rows / b) * math.exp(rng.uniform(-0.7, 0.7)))))
    j = max(1, rows // (b * i))
    i = min(i, max(1, rows // (b * j)))
    if op == "embed":
        v = rng.choice([21, 33, 66, 139, _log(rng, 2, 2048), _log(rng, 2048, 65536)])
        v = max(2, min(v, most // d))
        bins = rng.choice(["relpos", "padded", "uniform", "skewed"])
        return _embed(None, b, i, j, d, dtype, grad, v, rng.choice(["int32", "int64"]), bins, rng.random() < 0.5,
                      rng.choice([1.0, math.sqrt(d), 0.5]))
    p = rng.choice([0.1, 0.25, 0.25, 0.5]) if op == "dropout" else rng.choice([0.0, 0.0, 0.15, 0.25])
    layout = rng.choice(["whole", "whole", "block", "transposed"])
    residual = op == "dropout" or rng.random() < 0.75
    group = 0
    if op == "norm_fp8":
        group = rng.choice([g for g in (0, 32, 64, 128) if g == 0 or d % g == 0])
    return _pair(None, op, b, i, j, d, dtype, grad, p, rng.choice(["none", "rows", "columns"]), residual, layout, group)


def _generator(seed, salt):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) * 1000003 + salt)
    return g


def _view(case, seed, salt, scale):
    """A pair tensor of the case's layout: whole, a rank's block of a larger tensor, or a transposed view."""
    b, i, j, d, t = case["b"], case["i"], case["j"], case["d"], _TYPES[case["dtype"]]
    g = _generator(seed, salt)
    layout = case["layout"]
    shape = {"whole": (b, i, j, d), "block": (b, i + 1, j + 3, d), "transposed": (b, j, i, d)}[layout]
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    x = (x * scale).to(t)
    return x[:, 1:, 2:j + 2] if layout == "block" else x.transpose(1, 2) if layout == "transposed" else x


def prepare(case, seed):
    b, i, j, d, t = case["b"], case["i"], case["j"], case["d"], _TYPES[case["dtype"]]
    s = dict(case)
    g = _generator(seed, 1)
    if case["op"] == "embed":
        v, bins, kind = case["v"], case["bins"], {"int32": torch.int32, "int64": torch.int64}[case["index"]]
        if bins in ("relpos", "padded"):
            # clipped offsets between residues, with jumps between chains; "padded": no position behind the sequence's end
            at = torch.randint(0, 2, (b, max(i, j)), generator=g, device="cuda").mul_(7).add_(1).cumsum(1)
            half = max(1, (v - 2) // 2)
            index = (at[:, :i, None] - at[:, None, :j]).clamp(-half, half) + half
            index = index.clamp(0, v - 1)
            if bins == "padded":
                index[:, max(1, (9 * i) // 10):] = -1
                index[:, :, max(1, (9 * j) // 10):] = -1
        else:
            f = torch.rand((b, i, j), generator=g, device="cuda", dtype=torch.float32)
            index = ((f ** 6 if bins == "skewed" else f) * v).long().clamp(0, v - 1)
        s["index"] = index.to(kind)
        s["table"] = torch.randn((v, d), generator=g, device="cuda").mul_(0.1).to(t).requires_grad_(case["grad"])
        s["stream"] = torch.randn((b, i, j, d), generator=g, device="cuda").to(t).requires_grad_(case["grad"]) if case["base"] else None
        s["dout"] = torch.randn((b, i, j, d), generator=g, device="cuda").to(t) if case["grad"] else None
        return s
    s["update"] = _view(case, seed, 2, 0.5).requires_grad_(case["grad"])
    s["stream"] = _view(case, seed, 3, 2.0).requires_grad_(case["grad"]) if case["residual"] else None
    # this block's place in the whole grid, and the step's seed
    s["origin"] = (0, 5 * i, 3 * j)
    s["seed"], s["offset"] = (int(seed) * 0x9E3779B97F4A7C15 + 12345) % (1 << 63), int(seed) % 1000
    if case["op"] != "dropout":
        s["weight"] = (1 + 0.1 * torch.randn((d,), generator=g, device="cuda")).to(t).requires_grad_(case["grad"])
    if case["grad"]:
        s["dz"] = torch.randn((b, i, j, d), generator=g, device="cuda").to(t)
        if case["op"] == "norm":
            s["dy"] = torch.randn((b, i, j, d), generator=g, device="cuda").to(t)
    return s


# ------------------------------------------------------------------------------------------------
# the plain form
# ------------------------------------------------------------------------------------------------
def _keep(s):
    """Truth values of what the dropout keeps: Philox4x32-10 (Salmon et al., 2011) of the global position, 16 bits an element."""
    b, i, j, d, shared = s["b"], s["i"], s["j"], s["d"], s["shared"]
    b0, i0, j0 = s["origin"]
    dev = s["update"].device
    nv = (d + 7) // 8
    low = 0xFFFFFFFF

    def axis(n, start, dim):
        v = torch.arange(n, device=dev, dtype=torch.int64) + start
        return v.reshape([-1 if k == dim else 1 for k in range(4)])

    x0 = (axis(b, b0, 0) << 16) | axis(nv, 0, 3)
    x1 = axis(j, j0, 2) if shared != "columns" else torch.zeros((1, 1, 1, 1), dtype=torch.int64, device=dev)
    x2 = axis(i, i0, 1) if shared != "rows" else torch.zeros((1, 1, 1, 1), dtype=torch.int64, device=dev)
    x3 = torch.full((1, 1, 1, 1), s["offset"], dtype=torch.int64, device=dev)
    k0, k1 = s["seed"] & low, s["seed"] >> 32

    def rounds(x, k0, k1, left):
        if left == 0:
            return x
        p0, p1 = x[0] * 0xD2511F53, x[2] * 0xCD9E8D57
        return rounds((((p1 >> 32) & low) ^ x[1] ^ k0, p1 & low, ((p0 >> 32) & low) ^ x[3] ^ k1, p0 & low),
                      (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low, left - 1)

    words = torch.stack(torch.broadcast_tensors(*rounds((x0, x1, x2, x3), k0, k1, 10)), dim=-1)
    halves = torch.stack((words & 0xFFFF, words >> 16), dim=-1).reshape(*words.shape[:3], nv * 8)[..., :d]
    return halves < _threshold(s["p"])


def _threshold(p):
    return int(math.floor((1.0 - p) * 65536.0 + 0.5))


def _dropped(s, x, keep):
    return torch.where(keep, x * (65536.0 / _threshold(s["p"])), torch.zeros((), device=x.device, dtype=x.dtype))


def _plain_embed(s):
    t, v = s["table"].dtype, s["v"]
    index = s["index"].long()
    there = (index >= 0) & (index < v)
    row = torch.where(there, index, torch.zeros_like(index))
    out = torch.where(there[..., None], s["table"].float()[row], torch.zeros((), device=row.device)) * s["scale"]
    if s["stream"] is not None:
        out = out + s["stream"].float()
    out = out.to(t)
    if not s["grad"]:
        return out
    # sums over very many tokens: in 64 bits
    rows = torch.where(there, index, torch.full_like(index, v)).reshape(-1)
    sums = torch.zeros((v + 1, s["d"]), dtype=torch.float64, device=row.device)
    sums.index_add_(0, rows, s["dout"].reshape(-1, s["d"]).double())
    grads = [(sums[:v] * s["scale"]).to(t)]
    if s["stream"] is not None:
        grads.append(s["dout"])
    return [out] + grads


def _plain_pair(s):
    t, d = s["update"].dtype, s["d"]
    keep = _keep(s) if s["p"] > 0 else None
    u = s["update"].float()
    if keep is not None:
        u = _dropped(s, u, keep)
    z = (u if s["stream"] is None else u + s["stream"].float()).to(t)
    if s["op"] == "dropout":
        if not s["grad"]:
            return z
        return [z, _dropped(s, s["dz"].float(), keep).to(t), s["dz"]]
    # the norm reads the stream as it is stored
    zf, w = z.float(), s["weight"].float()
    r = torch.rsqrt(zf.square().mean(dim=-1, keepdim=True) + _EPS)
    y = zf * r * w
    if s["op"] == "norm_fp8":
        group = s["group"] or d
        yg = y.reshape(*y.shape[:3], d // group, group)
        most = yg.abs().amax(dim=-1, keepdim=True)
        scale = torch.where(most > 0, most / _E4M3_MAX, torch.ones_like(most))
        q = (yg / scale).reshape(y.shape).to(torch.float8_e4m3fn)
        return [q, scale.squeeze(-1), z]
    if not s["grad"]:
        return [y.to(t), z]
    dy, dz = s["dy"].float(), s["dz"].float()
    wdy = dy * w
    g = dz + r * wdy - zf * (r * r * r) * (wdy * zf).mean(dim=-1, keepdim=True)
    dw = (dy * zf * r).reshape(-1, d).sum(dim=0, dtype=torch.float64)
    du = g if keep is None else _dropped(s, g, keep)
    grads = [du.to(t)] + ([g.to(t)] if s["stream"] is not None else []) + [dw.to(t)]
    return [y.to(t), z] + grads


# ------------------------------------------------------------------------------------------------
# the framework's calls
# ------------------------------------------------------------------------------------------------
def _own(s):
    from fold_cp_ops_b200.workflows import pair_stream as P

    if s["op"] == "embed":
        out = P.pair_embedding(s["index"], s["table"], scale=s["scale"], base=s["stream"])
        if not s["grad"]:
            return out
        leaves = [s["table"]] + ([] if s["stream"] is None else [s["stream"]])
        return [out.detach(), *torch.autograd.grad(out, leaves, s["dout"])]
    drop = None
    if s["p"] > 0:
        drop = P.PairDropout(s["p"], seed=s["seed"], offset=s["offset"], shared=None if s["shared"] == "none" else s["shared"],
                             origin=s["origin"])
    leaves = [s["update"]] + ([] if s["stream"] is None else [s["stream"]])
    if s["op"] == "dropout":
        z = P.dropout_add(s["update"], s["stream"], drop)
        return [z.detach(), *torch.autograd.grad(z, leaves, s["dz"])] if s["grad"] else z
    if s["op"] == "norm_fp8":
        return list(P.add_rms_norm_fp8(s["update"], s["stream"], s["weight"], eps=_EPS, group=s["group"] or None, dropout=drop))
    y, z = P.add_rms_norm(s["update"], s["stream"], s["weight"], eps=_EPS, dropout=drop)
    if not s["grad"]:
        return [y, z]
    return [y.detach(), z.detach(), *torch.autograd.grad((y, z), leaves + [s["weight"]], (s["dy"], s["dz"]))]


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain_embed(state) if state["op"] == "embed" else _plain_pair(state)


def work(case):
    """Bytes: each input once, each output once.  Operations: the fp32 arithmetic of the formulas (the generator's integer
    work is not counted)."""
    rows, d, e, grad = case["b"] * case["i"] * case["j"], case["d"], _BYTES[case["dtype"]], case["grad"]
    n = rows * d
    if case["op"] == "embed":
        width = 4 if case["index"] == "int32" else 8
        tensors = 1 + (1 if case["base"] else 0) + (1 if grad else 0)
        table = min(rows, case["v"]) * d * e + (case["v"] * d * e if grad else 0)  # the rows looked up; all of the gradient
        return {"bytes": rows * width + tensors * n * e + table, "flops": n * (2 + (1 if grad else 0))}
    inputs = 1 + (1 if case["residual"] else 0)
    if case["op"] == "dropout":  # the residual's gradient is the output's: nothing to write
        return {"bytes": n * e * (inputs + 1 + (2 if grad else 0)), "flops": n * (2 + (1 if grad else 0))}
    stream = 1 if case["residual"] or case["p"] > 0 else 0  # otherwise the stream is the update itself
    if case["op"] == "norm_fp8":
        return {"bytes": n * e * (inputs + stream) + n + rows * 4 * (d // (case["group"] or d)) + d * e, "flops": 7 * n}
    size = n * e * (inputs + stream + 1) + d * e
    if grad:
        size += n * e * (4 if case["residual"] and case["p"] > 0 else 3) + d * e
    return {"bytes": size, "flops": n * (5 + (11 if grad else 0))}


# ------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def _mul_hi_lo(x, m):
    """High and low 32 bits of x * m from 16-bit limbs, so that no product passes 63 bits."""
    lo = x * (m & 0xFFFF)
    hi = x * (m >> 16) + (lo >> 16)
    return hi >> 16, ((hi & 0xFFFF) << 16) | (lo & 0xFFFF)


def _kept_exact(s):
    mask = (1 << 32) - 1
    grid = [torch.arange(n, device="cuda", dtype=torch.int64) for n in (s["b"], s["i"], s["j"], (s["d"] + 7) // 8)]
    cb, ci, cj, cv = torch.meshgrid(*grid, indexing="ij")
    ctr = [(cb + s["origin"][0]) * 65536 + cv, (cj + s["origin"][2]) * int(s["shared"] != "columns"),
           (ci + s["origin"][1]) * int(s["shared"] != "rows"), torch.full_like(cb, s["offset"])]
    key = [s["seed"] % (1 << 32), s["seed"] // (1 << 32)]
    for _ in range(10):
        (h0, l0), (h1, l1) = _mul_hi_lo(ctr[0], 0xD2511F53), _mul_hi_lo(ctr[2], 0xCD9E8D57)
        ctr = [h1 ^ ctr[1] ^ key[0], l1, h0 ^ ctr[3] ^ key[1], l0]
        key = [(key[0] + 0x9E3779B9) & mask, (key[1] + 0xBB67AE85) & mask]
    kept = torch.empty((s["b"], s["i"], s["j"], cv.shape[-1], 8), dtype=torch.bool, device="cuda")
    limit = round((1 - s["p"]) * 65536)
    for lane in range(8):
        kept[..., lane] = ((ctr[lane // 2] >> (16 * (lane % 2))) % 65536) < limit
    return kept.flatten(3)[..., :s["d"]], 65536 / limit


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "embed":
            return _exact_embed(s)
        t = s["update"].dtype
        u = s["update"].double()
        if s["p"] > 0:
            kept, gain = _kept_exact(s)
            u = (u * gain).masked_fill(~kept, 0.0)
        z = u if s["stream"] is None else u + s["stream"].double()
        if s["op"] == "dropout":
            if not s["grad"]:
                return z
            return [z, (s["dz"].double() * gain).masked_fill(~kept, 0.0), s["dz"].double()]
        stored = z.to(t).double()  # the norm is of the stream as it is stored
        w = s["weight"].double()
        norm = (stored.pow(2).sum(-1, keepdim=True) / s["d"] + _EPS).sqrt()
        unit = stored / norm
        y = unit * w
        if s["op"] == "norm_fp8":
            parts = y.unflatten(-1, (-1, s["group"] or s["d"]))
            top = parts.abs().max(dim=-1).values
            scale = torch.where(top == 0, torch.ones_like(top), top / _E4M3_MAX)
            return [(parts / scale[..., None]).flatten(3), scale, z]
        if not s["grad"]:
            return [y, z]
        dunit = s["dy"].double() * w
        g = s["dz"].double() + (dunit - unit * (dunit * unit).sum(-1, keepdim=True) / s["d"]) / norm
        dw = (s["dy"].double() * unit).sum(dim=(0, 1, 2))
        du = (g * gain).masked_fill(~kept, 0.0) if s["p"] > 0 else g
        return [y, z, du] + ([] if s["stream"] is None else [g]) + [dw]


def _exact_embed(s):
    v, d = s["v"], s["d"]
    flat = s["index"].reshape(-1).long()
    valid = (flat >= 0) & (flat < v)
    padded = torch.cat((s["table"].double() * s["scale"], torch.zeros((1, d), dtype=torch.float64, device="cuda")))
    slot = flat.masked_fill(~valid, v)
    out = padded.index_select(0, slot).reshape(*s["index"].shape, d)
    if s["stream"] is not None:
        out = s["stream"].double() + out
    if not s["grad"]:
        return out
    # sums of runs of the sorted tokens, from differences of a running sum
    order = torch.argsort(slot, stable=True)
    running = torch.cat((torch.zeros((1, d), dtype=torch.float64, device="cuda"),
                         s["dout"].reshape(-1, d)[order].double().cumsum(0)))
    ends = torch.searchsorted(slot[order], torch.arange(v + 1, device="cuda"))
    sums = running[ends[1:]] - running[ends[:-1]]
    return [out, sums * s["scale"]] + ([] if s["stream"] is None else [s["dout"].double()])
