"""Cases that measure the MXFP4 expert path and the fused block norms.

``run`` computes each operator in elementary torch operations, or, with ``own`` true, through the package's entry
points on the same inputs; ``exact`` gives the same outputs from the definitions in 64 bits.  Kinds of a case:

* ``mxfp4``        quantise a matrix to MXFP4 and read it back
* ``ffn``          the grouped SwiGLU experts of one layer on MXFP4 weights
* ``combine_norm`` weighted combine of the expert rows, post-norm, gate, residual, next block's pre-norm
* ``norm``         the same without the combine
"""
import math
import random

import torch

own = False

BLOCK = 32
EPS = 1e-6
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DTYPES = dict(bf16=torch.bfloat16, fp16=torch.float16, fp32=torch.float32)
SIZE = dict(bf16=2, fp16=2, fp32=4)

MAX_ELEMENTS = 128 * 768 * 2048          # largest matrix of the mxfp4 cases
MAX_WEIGHTS = 128 * 3 * 4096 * 1536      # largest layer of the ffn cases
MAX_ROW_FLOPS = 12450 * 8 * 2048 * 768   # rows * H * I of the prefill case


def listed():
    def q(name, rows, cols, dtype):
        return dict(name=name, kind="mxfp4", rows=rows, cols=cols, dtype=dtype)

    def f(name, tokens, hidden, inter, experts, top_k, skew=0.0):
        return dict(name=name, kind="ffn", tokens=tokens, hidden=hidden, inter=inter, experts=experts, top_k=top_k,
                    skew=skew)

    return [
        # one expert's gate projection, as an expert is converted when it is loaded
        q("quantise_expert", 768, 2048, "bf16"),
        # a ragged matrix of FP32 master weights
        q("quantise_ragged_fp32", 1007, 1056, "fp32"),
        # one projection of a whole layer's experts
        q("quantise_layer", 128 * 768, 2048, "bf16"),
        # one decode step of one user
        f("ffn_one_token", 1, 2048, 768, 128, 8),
        # a decode step at the serving batch
        f("ffn_decode_64", 64, 2048, 768, 128, 8),
        # sizes that no tile divides, a number of experts that is no power of two
        f("ffn_odd", 333, 1056, 416, 60, 4, skew=0.6),
        # a large decode batch of the larger model's layer
        f("ffn_large_256", 256, 4096, 1536, 128, 8),
        # a ragged prefill batch with a skewed router
        f("ffn_prefill", 12450, 2048, 768, 128, 8, skew=1.1),
        # between two layers of a decode step
        dict(name="combine_decode", kind="combine_norm", tokens=64, hidden=2048, top_k=8, post="rms", pre="rms",
             gate="none", act="none", residual="bf16"),
        # between two layers of a prefill step, with a gate for each token
        dict(name="combine_prefill", kind="combine_norm", tokens=12450, hidden=2048, top_k=8, post="rms", pre="rms",
             gate="token", act="sigmoid", residual="fp32"),
        # three tokens whose rows end inside a vector
        dict(name="norm_odd", kind="norm", tokens=3, hidden=5003, post="rms", pre="layer", gate="channel", act="none",
             residual="fp32"),
        # a prefill batch around a block that needs no combine
        dict(name="norm_prefill", kind="norm", tokens=12450, hidden=4096, post="layer", pre="rms", gate="full",
             act="sigmoid", residual="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("mxfp4", "ffn", "ffn", "combine_norm", "norm"))
    if kind == "mxfp4":
        cols = BLOCK * _log_int(rng, 1, 256)
        rows = _log_int(rng, 1, min(100000, MAX_ELEMENTS // (2 * cols)))
        return dict(kind=kind, rows=rows, cols=cols, dtype=rng.choice(("bf16", "fp16", "fp32")))
    if kind == "ffn":
        hidden = BLOCK * _log_int(rng, 4, 128)
        inter = BLOCK * _log_int(rng, 2, 48)
        experts = _log_int(rng, 1, min(256, MAX_WEIGHTS // (3 * hidden * inter)))
        top_k = rng.randint(1, min(8, experts))
        tokens = _log_int(rng, 1, max(1, min(12450, MAX_ROW_FLOPS // (top_k * hidden * inter))))
        return dict(kind=kind, tokens=tokens, hidden=hidden, inter=inter, experts=experts, top_k=top_k,
                    skew=rng.choice((0.0, 0.6, 1.1)))
    case = dict(kind=kind, tokens=_log_int(rng, 1, 12450), hidden=_log_int(rng, 16, 4096),
                post=rng.choice(("none", "rms", "layer")), pre=rng.choice(("none", "rms", "layer")),
                gate=rng.choice(("none", "token", "channel", "full")), act=rng.choice(("none", "sigmoid")),
                residual=rng.choice(("bf16", "fp32")))
    if kind == "combine_norm":
        case["top_k"] = rng.randint(1, 8)
        case["hidden"] = 8 * _log_int(rng, 2, 256)
    return case


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape, std=1.0):
    return torch.randn(*shape, device="cuda", generator=gen) * std


def _random_mxfp4(gen, experts, rows, cols):
    """Codes and scales of N(0, 0.02) weights, made directly in the quantised form: the largest of 32 normal values
    sets the block's exponent."""
    codes = torch.empty(experts, rows, cols // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(experts, rows, cols // BLOCK, dtype=torch.uint8, device="cuda")
    edges = torch.tensor([(a + b) / 2 for a, b in zip(E2M1, E2M1[1:])], device="cuda")
    step = max(1, (1 << 25) // (rows * cols))
    for e in range(0, experts, step):
        w = _normal(gen, min(step, experts - e), rows, cols // BLOCK, BLOCK, std=0.02)
        exp = torch.floor(torch.log2(w.abs().amax(-1, keepdim=True).clamp_min(1e-30))) - 2
        code = torch.bucketize(w.abs() * torch.exp2(-exp), edges, out_int32=True).to(torch.uint8)
        code |= (w < 0).to(torch.uint8) << 3
        code = code.view(-1, rows, cols)
        codes[e:e + step] = code[..., 0::2] | (code[..., 1::2] << 4)
        scales[e:e + step] = (exp.squeeze(-1) + 127).to(torch.uint8)
    return codes, scales


def _routing(case, seed):
    """Distinct experts for each token; the load of the experts is the case's, which expert has which load and
    which token comes where is the seed's."""
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    fixed = torch.Generator().manual_seed(t * 1000003 + e * 1009 + k)
    load = torch.arange(1, e + 1, dtype=torch.float64).pow(-case["skew"])
    ids = torch.topk(load.log() - torch.log(-torch.log(torch.rand(t, e, generator=fixed, dtype=torch.float64))),
                     k, dim=1).indices
    gen = torch.Generator().manual_seed(seed)
    ids = torch.randperm(e, generator=gen)[ids][torch.randperm(t, generator=gen)]
    return ids.contiguous()


def _inputs(case, seed):
    gen = _generator(seed)
    kind = case["kind"]
    if kind == "mxfp4":
        x = _normal(gen, case["rows"], case["cols"], std=0.02)
        return dict(x=x.to(DTYPES[case["dtype"]]))
    if kind == "ffn":
        h, i, e = case["hidden"], case["inter"], case["experts"]
        x = _normal(gen, case["tokens"], h)
        x[:, torch.randint(0, h, (max(1, h // 256),), device="cuda", generator=gen)] *= 8.0   # outlier channels
        s = dict(x=x.to(torch.bfloat16), ids=_routing(case, seed))
        for name, rows, cols in (("gate", i, h), ("up", i, h), ("down", h, i)):
            s[name] = _random_mxfp4(gen, e, rows, cols)
        flat = s["ids"].t().reshape(-1)                    # slot-major assignments, packed stably by expert
        s["counts"] = torch.bincount(flat, minlength=e).tolist()
        s["tokens"] = (torch.argsort(flat, stable=True) % case["tokens"]).cuda()
        return s
    t, h = case["tokens"], case["hidden"]
    bf = torch.bfloat16
    s = dict(residual=_normal(gen, t, h, std=2.0).to(DTYPES[case["residual"]]))
    if kind == "combine_norm":
        k = case["top_k"]
        s["rows"] = _normal(gen, t * k, h, std=0.5).to(bf)
        w = torch.rand(t, k, device="cuda", generator=gen) + 0.05
        s["weights"] = (w / w.sum(1, keepdim=True)).to(bf)
        s["inverse"] = torch.randperm(t * k, device="cuda", generator=gen).to(torch.int32)
    else:
        s["y"] = _normal(gen, t, h, std=0.5).to(bf)
    s["post_weight"] = (1 + _normal(gen, h, std=0.1)).to(bf) if case["post"] != "none" else None
    s["pre_weight"] = (1 + _normal(gen, h, std=0.1)).to(bf) if case["pre"] != "none" else None
    shape = dict(none=None, token=(t, 1), channel=(1, h), full=(t, h))[case["gate"]]
    s["gate"] = _normal(gen, *shape).to(bf) if shape else None
    s["residual_scale"], s["block_scale"] = 0.875, 1.25
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own and case["kind"] == "ffn":
        from pdscope_b200 import Mxfp4, Mxfp4ExpertSlab, pack
        ids = s["ids"].cuda()
        s["packed"] = pack(ids, torch.ones(ids.shape, dtype=torch.bfloat16, device="cuda"), case["experts"])
        s["slab"] = Mxfp4ExpertSlab.from_quantized(*(Mxfp4(*s[n]) for n in ("gate", "up", "down")))
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------


def _plain_quantise(x):
    b = x.float().view(*x.shape[:-1], -1, BLOCK)
    exp = (torch.frexp(b.abs().amax(-1, keepdim=True)).exponent - 3).clamp_min(-127)
    a = torch.ldexp(b.abs(), -exp)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (torch.round(a / step) * step).clamp_max(6.0)
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = (code | (torch.signbit(b).to(torch.uint8) << 3)).view(x.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), (exp.squeeze(-1) + 127).to(torch.uint8)


def _plain_dequantise(codes, scales):
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    v = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), -1)
    v = v.view(*codes.shape[:-1], -1, BLOCK)
    return torch.ldexp(v, scales.int().unsqueeze(-1) - 127).view(*codes.shape[:-1], -1)


def _plain_ffn(s):
    out = torch.empty(len(s["tokens"]), s["x"].shape[1], dtype=torch.bfloat16, device="cuda")
    a = 0
    for e, n in enumerate(s["counts"]):
        if n:
            g, u, d = (_plain_dequantise(s[m][0][e], s[m][1][e]) for m in ("gate", "up", "down"))
            x = s["x"][s["tokens"][a:a + n]].float()
            h = x @ g.t()
            h = h * torch.sigmoid(h) * (x @ u.t())
            out[a:a + n] = (h @ d.t()).to(torch.bfloat16)
            a += n
    return out


def _plain_norm(v, how, weight):
    if how == "none":
        return v
    if how == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * torch.rsqrt((v * v).mean(-1, keepdim=True) + EPS)
    return v if weight is None else v * weight.float()


def _plain_block(s, y):
    case = s["case"]
    z = _plain_norm(y, case["post"], s["post_weight"])
    if s["gate"] is not None:
        g = s["gate"].float()
        z = z * (torch.sigmoid(g) if case["act"] == "sigmoid" else g)
    r = s["residual_scale"] * s["residual"].float() + s["block_scale"] * z
    n = _plain_norm(r, case["pre"], s["pre_weight"])
    return r.to(s["residual"].dtype), n.to(torch.bfloat16)


def run(s):
    case = s["case"]
    kind = case["kind"]
    if own:
        import pdscope_b200 as pdx
        if kind == "mxfp4":
            return pdx.dequantize_mxfp4(pdx.quantize_mxfp4(s["x"]), s["x"].dtype)
        if kind == "ffn":
            return pdx.moe_ffn_mxfp4(s["x"], s["packed"], s["slab"])
        options = dict(post=case["post"], post_weight=s["post_weight"], gate=s["gate"], gate_act=case["act"],
                       residual_scale=s["residual_scale"], block_scale=s["block_scale"], pre=case["pre"],
                       pre_weight=s["pre_weight"], eps=EPS)
        if kind == "norm":
            return pdx.block_norm(s["y"], s["residual"], **options)
        return pdx.combine_block_norm(s["rows"], s["weights"], s["inverse"], s["residual"], **options)
    if kind == "mxfp4":
        return _plain_dequantise(*_plain_quantise(s["x"])).to(s["x"].dtype)
    if kind == "ffn":
        return _plain_ffn(s)
    if kind == "norm":
        return _plain_block(s, s["y"].float())
    t, k = s["weights"].shape
    y = s["rows"][s["inverse"].view(t, k).long()].float()
    return _plain_block(s, (y * s["weights"].float().unsqueeze(-1)).sum(1))


# ---------------------------------------------------------------------------
# The same from the definitions in 64 bits
# ---------------------------------------------------------------------------


def _exact_weight(codes, scales):
    """E2M1: (-1)^s 2^(max(e, 1) - 1) (m/2 + (e > 0)), times 2^(scale - 127)."""
    c = torch.empty(codes.shape[0], codes.shape[1] * 2, dtype=torch.int32, device=codes.device)
    c[:, 0::2], c[:, 1::2] = codes & 15, codes >> 4
    e, m = (c >> 1) & 3, (c & 1).double()
    v = torch.pow(2.0, (e.clamp_min(1) - 1).double()) * (m / 2 + (e > 0).double()) * (1 - 2 * (c >> 3)).double()
    return v * torch.pow(2.0, scales.double() - 127).repeat_interleave(BLOCK, dim=1)


def _exact_mxfp4(x):
    grid = torch.tensor(E2M1, dtype=torch.float64, device="cuda")
    out = torch.empty(x.shape, dtype=torch.float64, device="cuda")
    for a in range(0, x.shape[0], 4096):
        b = x[a:a + 4096].double().view(-1, x.shape[1] // BLOCK, BLOCK)
        big = b.abs().amax(-1, keepdim=True)
        low = torch.where(big > 0, torch.floor(torch.log2(big)), -125.0) - 2
        unit = torch.pow(2.0, low.clamp_min(-127.0))
        mag = (b.abs() / unit).clamp_max(6.0)
        hi = torch.searchsorted(grid, mag.contiguous()).clamp_max(7)     # first grid value >= mag
        lo = (hi - 1).clamp_min(0)
        up, down = grid[hi] - mag, mag - grid[lo]
        pick = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)   # ties to the even code
        out[a:a + 4096] = (torch.sign(b) * grid[pick] * unit).view(-1, x.shape[1])
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "mxfp4":
        return _exact_mxfp4(s["x"])
    if kind == "ffn":
        parts, start = [], 0
        for e, n in enumerate(s["counts"]):
            if not n:
                continue
            x = s["x"].double().index_select(0, s["tokens"][start:start + n])
            g = torch.mm(x, _exact_weight(s["gate"][0][e], s["gate"][1][e]).t())
            u = torch.mm(x, _exact_weight(s["up"][0][e], s["up"][1][e]).t())
            parts.append(torch.mm(g / (1 + torch.exp(-g)) * u, _exact_weight(s["down"][0][e], s["down"][1][e]).t()))
            start += n
        return torch.cat(parts)
    if kind == "norm":
        y = s["y"].double()
    else:
        y = torch.zeros(s["residual"].shape, dtype=torch.float64, device="cuda")
        inverse = s["inverse"].view(s["weights"].shape).long()
        for j in range(inverse.shape[1]):
            y += s["weights"][:, j:j + 1].double() * s["rows"][inverse[:, j]].double()

    def norm(v, how, weight):
        if how == "none":
            return v
        center = v.mean(1, keepdim=True) if how == "layer" else 0.0
        spread = torch.sqrt(((v - center) ** 2).sum(1, keepdim=True) / v.shape[1] + EPS)
        return (v - center) / spread * weight.double()

    z = norm(y, case["post"], s["post_weight"])
    if s["gate"] is not None:
        g = s["gate"].double()
        z = z * (1 / (1 + torch.exp(-g)) if case["act"] == "sigmoid" else g)
    r = s["residual_scale"] * s["residual"].double() + s["block_scale"] * z
    return r, norm(r, case["pre"], s["pre_weight"])


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind == "mxfp4":
        n = case["rows"] * case["cols"]
        # the matrix read, its values written; codes and scales written by one and read by the other
        return dict(bytes=n * 2 * SIZE[case["dtype"]] + 2 * (n // 2 + n // BLOCK), flops=4 * n)
    t, h = case["tokens"], case["hidden"]
    if kind == "ffn":
        k, i = case["top_k"], case["inter"]
        active = len(set(_routing(case, 0).view(-1).tolist()))
        weights = active * (3 * h * i // 2 + 3 * h * i // BLOCK)
        return dict(bytes=weights + t * h * 2 + t * k * (4 + h * 2), flops=6 * t * k * h * i)
    res = SIZE[case["residual"]]
    gate = dict(none=0, token=t, channel=h, full=t * h)[case["gate"]] * 2
    norms = ((case["post"] != "none") + (case["pre"] != "none")) * h * 2
    rows = case.get("top_k", 1)
    extra = t * rows * 6 if kind == "combine_norm" else 0
    return dict(bytes=t * h * (2 * rows + 2 * res + 2) + gate + norms + extra, flops=t * h * (2 * rows + 12))


if __name__ == "__main__":
    for c in listed() + [draw(random.Random(0))]:
        print(c, work(c))
