"""The fused block norms against their 64-bit definition, alone and inside a
stack of MoE blocks."""
import numpy as np
import pytest
import torch

from tests import mxfp4_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def pdx():
    import pdscope_b200
    return pdscope_b200


def _f64(t):
    return None if t is None else t.double().cpu().numpy()


def _inputs(tokens, hidden, residual, gate, seed, offset=0.0):
    gen = torch.Generator().manual_seed(seed)
    bf = torch.bfloat16
    t = dict(y=(torch.randn(tokens, hidden, generator=gen) + offset).to(bf),
             residual=(2 * torch.randn(tokens, hidden, generator=gen) - offset).to(residual),
             post_weight=(1 + 0.2 * torch.randn(hidden, generator=gen)).to(bf),
             pre_weight=(1 + 0.2 * torch.randn(hidden, generator=gen)).to(bf))
    shape = dict(none=None, scalar=(), token=(tokens, 1), channel=(hidden,), row=(1, hidden),
                 full=(tokens, hidden))[gate]
    t["gate"] = torch.randn(shape, generator=gen).to(bf) if shape is not None else None
    return {k: (v.cuda() if v is not None else None) for k, v in t.items()}


def _check(got, y, residual, options):
    """FP32 sums of up to 8192 values in at most 32 + 8 + 5 steps are off by
    under 2^-18 of the sum of magnitudes, and each element sees a dozen more
    roundings: 2^-17 of the magnitudes in front of each rounding covers both.
    A centred value is off by 2^-17 of the row's largest."""
    o = {k: (_f64(v) if isinstance(v, torch.Tensor) else v) for k, v in options.items()}
    s, n = ref.block_norm(y, residual, **o)
    eps = o.get("eps", 1e-6)

    def gain(v, how, w):
        if how == "none":
            return np.ones_like(v)
        c = v - v.mean(-1, keepdims=True) if how == "layer" else v
        return np.abs(np.ones_like(v) if w is None else w) / np.sqrt((c * c).mean(-1, keepdims=True) + eps)

    ds = 2.0 ** -17 * np.abs(o.get("residual_scale", 1.0) * residual)
    if y is not None:
        g = 1.0 if o.get("gate") is None else np.abs(o["gate"])
        if o.get("gate_act") == "sigmoid" and o.get("gate") is not None:
            g = 1 / (1 + np.exp(-o["gate"]))
        lift = gain(y, o.get("post", "none"), o.get("post_weight")) * np.abs(y).max(-1, keepdims=True)
        ds = ds + 2.0 ** -17 * np.abs(o.get("block_scale", 1.0)) * g * lift
    half = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
    stream, normed = got
    err = np.abs(_f64(stream) - s)
    assert (err <= half[stream.dtype] * (np.abs(s) + ds) + ds + 1e-38).all()
    up = gain(s, o.get("pre", "rms"), o.get("pre_weight"))
    dn = up * (2 * ds.max(-1, keepdims=True) + 2.0 ** -17 * np.abs(s).max(-1, keepdims=True))
    err = np.abs(_f64(normed) - n)
    assert (err <= 2.0 ** -8 * (np.abs(n) + dn) + dn + 1e-38).all()


@pytest.mark.parametrize("tokens,hidden", ((1, 1), (3, 7), (2, 8), (5, 1003), (4, 1032), (33, 2048), (1, 4096), (2, 5003),
                                           (3, 8192), (300, 96), (700, 1), (700, 13), (700, 260), (601, 2041), (600, 4099),
                                           (597, 8175), (597, 8190)))
@pytest.mark.parametrize("residual", (torch.bfloat16, torch.float32))
@pytest.mark.parametrize("post,pre,gate,act", (("rms", "rms", "none", "none"), ("layer", "rms", "token", "sigmoid"),
                                               ("none", "layer", "channel", "none"), ("rms", "none", "full", "sigmoid"),
                                               ("layer", "layer", "row", "none"), ("none", "none", "scalar", "none")))
def test_block_norm(pdx, tokens, hidden, residual, post, pre, gate, act):
    t = _inputs(tokens, hidden, residual, gate, seed=tokens * 10000 + hidden)
    options = dict(post=post, pre=pre, gate=t["gate"], gate_act=act, residual_scale=0.75, block_scale=-1.5,
                   post_weight=t["post_weight"] if post != "none" else None,
                   pre_weight=t["pre_weight"] if pre != "none" else None)
    got = pdx.block_norm(t["y"], t["residual"], **options)
    assert got[0].dtype == residual and got[1].dtype == torch.bfloat16
    _check(got, _f64(t["y"]), _f64(t["residual"]), options)


def test_defaults_no_weights_and_offset(pdx):
    t = _inputs(6, 640, torch.float32, "none", seed=1, offset=30.0)
    for options in ({}, dict(post="layer", pre="layer"), dict(post="rms", eps=1e-2)):
        _check(pdx.block_norm(t["y"], t["residual"], **options), _f64(t["y"]), _f64(t["residual"]), options)
    got = pdx.block_norm(None, t["residual"], pre_weight=t["pre_weight"], residual_scale=2.0)
    _check(got, None, _f64(t["residual"]), dict(pre_weight=t["pre_weight"], residual_scale=2.0))


def test_zero_rows_and_non_finite_rows(pdx):
    """A zero row gives a zero row (eps keeps the norm finite); a row with NaN or
    infinity spoils itself alone."""
    t = _inputs(5, 264, torch.bfloat16, "none", seed=2)
    clean = pdx.block_norm(t["y"], t["residual"], post="rms")
    t["y"][1], t["residual"][1] = 0, 0
    t["y"][3, 5], t["y"][4, 6] = float("nan"), float("inf")
    s, n = pdx.block_norm(t["y"], t["residual"], post="rms")
    assert (s[1] == 0).all() and (n[1] == 0).all()
    assert n[3].isnan().all() and n[4].isnan().any()
    for i in (0, 2):
        assert torch.equal(s[i], clean[0][i]) and torch.equal(n[i], clean[1][i])


@pytest.mark.parametrize("hidden", (256, 257))
def test_strided_gates_and_aliased_outputs(pdx, hidden):
    t = _inputs(9, hidden, torch.bfloat16, "none", seed=3)
    wide = torch.randn(18, 2 * hidden + 3, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    for gate in (wide[::2, :hidden], wide[:9, 1:hidden + 1], wide[:9, : 2 * hidden: 2],
                 wide.t()[:hidden, :9].t(), wide[:9, :1]):
        options = dict(post="rms", gate=gate, gate_act="sigmoid")
        _check(pdx.block_norm(t["y"], t["residual"], **options), _f64(t["y"]), _f64(t["residual"]), options)
    want = pdx.block_norm(t["y"], t["residual"], post="rms")
    y, r = t["y"].clone(), t["residual"].clone()
    got = pdx.block_norm(y, r, post="rms", stream_out=r, out=y)
    assert got[0] is r and got[1] is y
    assert torch.equal(r, want[0]) and torch.equal(y, want[1])


def test_overlapping_outputs_are_refused(pdx):
    t = _inputs(4, 64, torch.bfloat16, "full", seed=3)
    both = torch.zeros(5, 64, dtype=torch.bfloat16, device="cuda")
    wide = torch.zeros(4, 64, dtype=torch.float32, device="cuda")
    half = wide.view(-1)[:128].view(torch.bfloat16).view(4, 64)     # BF16 over the first half of an FP32 stream
    for kw, match in ((dict(stream_out=both[:4], out=both[1:]), "must not overlap"),
                      (dict(y=both[1:], out=both[:4]), "lie apart"),
                      (dict(residual=wide, out=half), "lie apart"),
                      (dict(out=t["gate"]), "gate")):
        args = dict(dict(y=t["y"], residual=t["residual"]), **kw)
        with pytest.raises(ValueError, match=match):
            pdx.block_norm(args.pop("y"), args.pop("residual"), gate=t["gate"], **args)
    rows = torch.zeros(8, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="expert rows"):
        pdx.combine_block_norm(rows, torch.ones(4, 2, dtype=torch.bfloat16, device="cuda"),
                               torch.arange(8, dtype=torch.int32, device="cuda"), t["residual"], out=rows[4:])


@pytest.mark.parametrize("tokens,hidden,top_k", ((1, 64, 1), (1, 2048, 8), (7, 1003, 3), (64, 2048, 8), (5, 4096, 12),
                                                 (3, 8192, 32)))
@pytest.mark.parametrize("residual", (torch.bfloat16, torch.float32))
def test_combine_block_norm(pdx, tokens, hidden, top_k, residual):
    t = _inputs(tokens, hidden, residual, "token", seed=hidden + top_k)
    gen = torch.Generator().manual_seed(tokens)
    rows = torch.randn(tokens * top_k, hidden, generator=gen).to(torch.bfloat16).cuda()
    weights = torch.rand(tokens, top_k, generator=gen).to(torch.bfloat16).cuda()
    inverse = torch.randperm(tokens * top_k, generator=gen).to(torch.int32).cuda()
    options = dict(post="rms", post_weight=t["post_weight"], gate=t["gate"], gate_act="sigmoid", pre_weight=t["pre_weight"])
    got = pdx.combine_block_norm(rows, weights, inverse, t["residual"], **options)
    y = (_f64(rows)[inverse.cpu().numpy()].reshape(tokens, top_k, hidden) * _f64(weights)[..., None])
    # the FP32 combine is off by top_k 2^-24 of the magnitudes, inside _check's 2^-17 of the row's largest
    _check(got, y.sum(1), _f64(t["residual"]), options)


def test_combine_flags_rows_out_of_range(pdx):
    from pdscope_b200 import runtime
    t = _inputs(2, 64, torch.bfloat16, "none", seed=8)
    rows = torch.randn(4, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    weights = torch.ones(2, 2, dtype=torch.bfloat16, device="cuda")
    good = pdx.combine_block_norm(rows, weights, torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda"),
                                  t["residual"])
    got = pdx.combine_block_norm(rows, weights, torch.tensor([0, 1, 2, 4], dtype=torch.int32, device="cuda"),
                                 t["residual"])
    with pytest.raises(ValueError, match="expert ID"):
        runtime.raise_device_error()
    assert torch.equal(got[0][0], good[0][0])
    assert got[0].isfinite().all()


@pytest.mark.parametrize("mx", (False, True))
@pytest.mark.parametrize("residual", (torch.bfloat16, torch.float32))
@pytest.mark.parametrize("tokens", (1, 20, 90))
def test_stack_of_blocks(pdx, mx, residual, tokens):
    """A pre-norm stack on BF16 and on MXFP4 experts: the fused step, its graph
    and the staged path agree with the parts run one by one."""
    from pdscope_b200.stack import ResidentMoEStack
    layers, hidden, inter, experts, k = 3, 256, 128, 8, 2
    gen = torch.Generator(device="cuda").manual_seed(5)
    gates = [(torch.randn(experts, hidden, device="cuda", generator=gen) * 0.05).to(torch.bfloat16)
             for _ in range(layers)]
    slabs = [pdx.ExpertSlab.allocate(experts, hidden, inter, "cuda", std=0.1, generator=gen) for _ in range(layers)]
    if mx:
        slabs = [pdx.Mxfp4ExpertSlab.from_slab(s) for s in slabs]
    bf = torch.bfloat16
    norms = [pdx.BlockNorm(post="rms", pre="rms", residual_scale=0.9, block_scale=0.5,
                           post_weight=(1 + 0.1 * torch.randn(hidden, device="cuda", generator=gen)).to(bf),
                           pre_weight=(1 + 0.1 * torch.randn(hidden, device="cuda", generator=gen)).to(bf))
             for _ in range(layers + 1)]
    norms[2].gate, norms[2].gate_act = torch.randn(hidden, device="cuda", generator=gen).to(bf), "sigmoid"
    stack = ResidentMoEStack(gates, slabs, top_k=k, norms=norms, residual_dtype=residual)
    x = torch.randn(tokens, hidden, device="cuda", generator=gen).to(residual)
    stack.input(tokens).copy_(x)
    s, n = pdx.block_norm(None, x, norm=norms[0])
    for l in range(layers):
        r = pdx.route(n, gates[l], k, True)
        packed = pdx.pack(r.selected, r.weights, experts)
        if mx:
            rows = pdx.moe_ffn_mxfp4(n, packed, slabs[l])
        else:
            from pdscope_b200 import runtime
            rows = torch.empty(tokens * k, hidden, dtype=bf, device="cuda")
            ws = torch.empty(runtime.ffn_workspace_bytes(slabs[l], tokens * k, experts), dtype=torch.uint8, device="cuda")
            runtime.grouped_ffn(n, tokens, packed.tokens, packed.offsets, packed.active, experts, tokens * k, slabs[l],
                                rows, ws)
        s, n = pdx.combine_block_norm(rows, r.weights, packed.inverse, s, norm=norms[l + 1])
    for run in (lambda: stack.step(tokens, graph=False), lambda: stack.step(tokens), lambda: stack.step(tokens),
                lambda: stack.stage_once(tokens)):
        stack.output(tokens).zero_()
        run()
        assert torch.equal(stack.output(tokens), n) and torch.equal(stack.residual(tokens), s)
    stack.release_graphs()


@pytest.mark.parametrize("tokens", (1, 40))
def test_two_layer_protocol_on_mxfp4(pdx, tokens):
    """Without norms an MXFP4 stack runs the two-layer protocol of the BF16 one."""
    from pdscope_b200.stack import ResidentMoEStack
    from pdscope_b200.runtime import residual_layernorm
    gen = torch.Generator(device="cuda").manual_seed(6)
    gates = [(torch.randn(8, 256, device="cuda", generator=gen) * 0.05).to(torch.bfloat16) for _ in range(2)]
    slabs = [pdx.Mxfp4ExpertSlab.from_slab(pdx.ExpertSlab.allocate(8, 256, 128, "cuda", std=0.1, generator=gen))
             for _ in range(2)]
    stack = ResidentMoEStack(gates, slabs, top_k=2)
    x = torch.randn(tokens, 256, device="cuda", generator=gen).to(torch.bfloat16)
    stack.input(tokens).copy_(x)
    stack.step(tokens)
    for gate, slab in zip(gates, slabs):
        x = residual_layernorm(pdx.ResidentMoELayer(gate, slab, top_k=2).forward(x).out, x)
    assert torch.equal(stack.output(tokens), x)
    stack.release_graphs()


def _norm_stack(pdx, layers=2, hidden=128, experts=4, mx=True, seed=5):
    from pdscope_b200.stack import ResidentMoEStack
    gen = torch.Generator(device="cuda").manual_seed(seed)
    gates = [(torch.randn(experts, hidden, device="cuda", generator=gen) * 0.05).to(torch.bfloat16)
             for _ in range(layers)]
    slabs = [pdx.ExpertSlab.allocate(experts, hidden, 64, "cuda", std=0.1, generator=gen) for _ in range(layers)]
    if mx:
        slabs = [pdx.Mxfp4ExpertSlab.from_slab(s) for s in slabs]
    norms = [pdx.BlockNorm(post="rms", residual_scale=0.9, block_scale=0.5) for _ in range(layers + 1)]
    return ResidentMoEStack(gates, slabs, top_k=2, norms=norms)


def _both(stack, tokens):
    """Outputs of the captured step and of the step without a graph."""
    got = []
    for graph in (True, False):
        stack.output(tokens).zero_()
        stack.residual(tokens).zero_()
        stack.step(tokens, graph=graph)
        got.append((stack.output(tokens).clone(), stack.residual(tokens).clone()))
    return got


@pytest.mark.parametrize("mx", (False, True))
def test_captured_step_follows_its_norms(pdx, mx):
    """Scales, norm kinds, eps, weights and gates changed between two steps: the
    captured step gives what the step without a graph gives."""
    stack, tokens = _norm_stack(pdx, mx=mx), 6
    gen = torch.Generator(device="cuda").manual_seed(1)
    stack.input(tokens).copy_(torch.randn(tokens, 128, device="cuda", generator=gen))
    vector = lambda *shape: torch.randn(*shape, device="cuda", generator=gen).to(torch.bfloat16)
    kept = [vector(tokens, 1), vector(tokens, 1), vector(tokens, 128)]      # all alive throughout
    changes = [None, dict(residual_scale=0.5), dict(block_scale=-2.0), dict(pre="layer"), dict(post="none"),
               dict(post="layer", eps=0.5), dict(pre_weight=vector(128)), dict(pre_weight=vector(128)),
               dict(gate=kept[0]), dict(gate=kept[1]), dict(gate_act="sigmoid"), dict(gate=kept[2]),
               dict(gate=kept[2][:, :1]), dict(gate=kept[2][0]), dict(gate=None)]
    previous = None
    for change in changes:
        for name, value in (change or {}).items():
            setattr(stack.norms[1], name, value)
        graph, eager = _both(stack, tokens)
        assert torch.equal(graph[0], eager[0]) and torch.equal(graph[1], eager[1]), change
        assert previous is None or not torch.equal(eager[0], previous) or change == dict(gate_act="sigmoid"), change
        previous = eager[0]
    stack.norms[0] = pdx.BlockNorm(residual_scale=3.0, pre="none")
    graph, eager = _both(stack, tokens)
    assert torch.equal(graph[0], eager[0]) and torch.equal(graph[1], eager[1])
    stack.release_graphs()


def test_captured_step_keeps_its_gates(pdx):
    """A gate replaced every step, the old one dropped: each step reads its own.
    A gate written in place needs no new capture."""
    stack, tokens = _norm_stack(pdx), 6
    gen = torch.Generator(device="cuda").manual_seed(1)
    stack.input(tokens).copy_(torch.randn(tokens, 128, device="cuda", generator=gen))
    for i in range(4):
        stack.norms[1].gate = torch.randn(tokens, 1, device="cuda", generator=gen).to(torch.bfloat16)
        stack.step(tokens)
        got = stack.output(tokens).clone()
        junk = [torch.full((tokens, 1), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(8)]
        stack.step(tokens)
        stack.step(tokens, graph=False)
        assert torch.equal(got, stack.output(tokens)), i
        del junk
    stack.step(tokens)
    graphs = dict(stack._graphs)
    stack.norms[1].gate.fill_(0.25)
    graph, eager = _both(stack, tokens)
    assert torch.equal(graph[0], eager[0]) and not torch.equal(graph[0], got)
    assert stack._graphs == graphs and len(graphs) == 1
    stack.release_graphs()


def test_captured_step_refuses_bad_norms(pdx):
    """A norm that no longer fits is refused, not replayed from the capture; set
    right again, the step runs."""
    stack, tokens = _norm_stack(pdx), 6
    stack.input(tokens).fill_(0.5)
    stack.step(tokens)
    want = stack.output(tokens).clone()
    good = stack.norms[1]
    for bad in (dict(gate=torch.zeros(5, 1, dtype=torch.bfloat16, device="cuda")), dict(post="batch"), dict(eps=0.0),
                dict(pre_weight=torch.ones(64, dtype=torch.bfloat16, device="cuda"))):
        stack.norms[1] = pdx.BlockNorm(**dict(dict(post="rms", residual_scale=0.9, block_scale=0.5), **bad))
        with pytest.raises(ValueError):
            stack.step(tokens)
        stack.norms[1] = good
        stack.output(tokens).zero_()
        stack.step(tokens)
        assert torch.equal(stack.output(tokens), want)
    stack.release_graphs()


@pytest.mark.parametrize("tokens", (4, 700))
@pytest.mark.parametrize("hidden", (264, 1003))
def test_without_a_block_its_terms_do_not_apply(pdx, tokens, hidden):
    """y = None: neither the gate nor the block scale enters, whatever they hold."""
    t = _inputs(tokens, hidden, torch.float32, "full", seed=5)
    t["gate"][0, 1], t["gate"][1, 2], t["gate"][2, 3] = float("inf"), float("nan"), float("-inf")
    options = dict(pre_weight=t["pre_weight"], residual_scale=0.5)
    want = pdx.block_norm(None, t["residual"], **options)
    _check(want, None, _f64(t["residual"]), options)
    for extra in (dict(gate=t["gate"]), dict(gate=t["gate"], gate_act="sigmoid"), dict(gate=t["gate"][1, 2]),
                  dict(block_scale=float("inf")), dict(block_scale=float("nan"), post="layer")):
        got = pdx.block_norm(None, t["residual"], **options, **extra)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), list(extra)


@pytest.mark.parametrize("mx", (False, True))
@pytest.mark.parametrize("with_norms", (False, True))
@pytest.mark.parametrize("inters", ((128, 320), (320, 96, 128)))
def test_stack_of_experts_of_several_sizes(pdx, mx, with_norms, inters):
    """Layers whose experts differ in I: the fused step, its graph and the staged path agree with single layers."""
    from pdscope_b200.runtime import residual_layernorm
    from pdscope_b200.stack import ResidentMoEStack
    gen = torch.Generator(device="cuda").manual_seed(8)
    experts, hidden, tokens = 4, 256, 9
    gates = [(torch.randn(experts, hidden, device="cuda", generator=gen) * 0.05).to(torch.bfloat16) for _ in inters]
    slabs = [pdx.ExpertSlab.allocate(experts, hidden, i, "cuda", std=0.1, generator=gen) for i in inters]
    if mx:
        slabs = [pdx.Mxfp4ExpertSlab.from_slab(s) for s in slabs]
    norms = [pdx.BlockNorm(post="rms") for _ in range(len(inters) + 1)] if with_norms else None
    stack = ResidentMoEStack(gates, slabs, top_k=2, norms=norms)
    x = torch.randn(tokens, hidden, device="cuda", generator=gen).to(torch.bfloat16)
    stack.input(tokens).copy_(x)
    stack.stage_once(tokens)
    want = stack.output(tokens).clone()
    if not with_norms:
        for gate, slab in zip(gates, slabs):
            x = residual_layernorm(pdx.ResidentMoELayer(gate, slab, top_k=2).forward(x).out, x)
        assert torch.equal(want, x)
    for graph in (False, True):
        stack.output(tokens).zero_()
        stack.step(tokens, graph=graph)
        assert torch.equal(stack.output(tokens), want)
    stack.release_graphs()


def test_layer_and_runtime_refuse_short_slabs(pdx):
    """Slabs whose slots or slot table do not cover the router's experts, or of another hidden size."""
    gate = torch.zeros(4, 64, dtype=torch.bfloat16, device="cuda")
    x = torch.zeros(2, 64, dtype=torch.bfloat16, device="cuda")
    short = torch.zeros(3, dtype=torch.int32, device="cuda")
    storage = torch.zeros(4 * 3 * 64 * 64, dtype=torch.bfloat16, device="cuda")
    for slab in (pdx.Mxfp4ExpertSlab(3, 64, 64, "cuda"), pdx.Mxfp4ExpertSlab(4, 64, 64, "cuda", slot_of_expert=short),
                 pdx.ExpertSlab(storage, 64, 64, slot_of_expert=short)):
        with pytest.raises(ValueError, match="fewer experts"):
            pdx.ResidentMoELayer(gate, slab)
        with pytest.raises(ValueError, match="fewer experts"):
            pdx.PDScopeCudaRuntime({0: slab}, top_k=2).forward(x, gate, layer=0, step=0, top_k=2)
    wide = pdx.Mxfp4ExpertSlab(4, 128, 64, "cuda")
    with pytest.raises(ValueError, match="hidden"):
        pdx.PDScopeCudaRuntime({0: wide}, top_k=2).forward(x, gate, layer=0, step=0, top_k=2)


def test_outputs_over_weights_are_refused(pdx):
    """Every row reads the weights, the combine's weights and its order: no output may lie over them."""
    t = _inputs(4, 64, torch.bfloat16, "none", seed=3)
    out = torch.ones(4, 64, dtype=torch.bfloat16, device="cuda")
    wide = torch.ones(4, 64, dtype=torch.float32, device="cuda")
    for kw in (dict(out=out, pre_weight=out[2]), dict(stream_out=out, post="rms", post_weight=out[0])):
        with pytest.raises(ValueError, match="weights"):
            pdx.block_norm(t["y"], t["residual"], **kw)
    rows = torch.zeros(8, 64, dtype=torch.bfloat16, device="cuda")
    weights, order = torch.ones(4, 2, dtype=torch.bfloat16, device="cuda"), torch.arange(8, dtype=torch.int32, device="cuda")
    for args, kw in (((out.view(-1)[:8].view(4, 2), order, t["residual"]), dict(out=out)),
                     ((weights, wide.view(torch.int32).view(-1)[:8], wide.clone()), dict(stream_out=wide)),
                     ((weights, order, t["residual"]), dict(stream_out=out, pre_weight=out[3]))):
        with pytest.raises(ValueError, match="weights"):
            pdx.combine_block_norm(rows, *args, **kw)
    with pytest.raises(ValueError):
        pdx.block_norm(t["y"], t["residual"], out=out, pre_weight=[1.0] * 64)


# From 593 rows on other kernels run than for few: two vectors a thread (256 threads to H = 4096, 512 beyond), or
# value by value (256 threads to H = 2048, 512 to 4096), with the weights and beside expert rows the gate loaded late.
MANY_ROWS = ((593, 8), (601, 264), (700, 2048), (595, 4096), (593, 4104), (600, 8192),       # vectors
             (593, 9), (600, 2047), (601, 2049), (593, 3001), (594, 4095), (593, 5001))      # value by value


@pytest.mark.parametrize("tokens,hidden", MANY_ROWS)
@pytest.mark.parametrize("residual", (torch.bfloat16, torch.float32))
@pytest.mark.parametrize("post,pre,gate,act", (("rms", "rms", "none", "none"), ("layer", "rms", "full", "sigmoid"),
                                               ("none", "layer", "channel", "none"), ("rms", "none", "token", "sigmoid"),
                                               ("layer", "layer", "full", "none")))
def test_many_rows(pdx, tokens, hidden, residual, post, pre, gate, act):
    t = _inputs(tokens, hidden, residual, gate, seed=tokens * 10000 + hidden)
    options = dict(post=post, pre=pre, gate=t["gate"], gate_act=act, residual_scale=0.75, block_scale=-1.5,
                   post_weight=t["post_weight"] if post != "none" else None,
                   pre_weight=t["pre_weight"] if pre != "none" else None)
    want = pdx.block_norm(t["y"], t["residual"], **options)
    _check(want, _f64(t["y"]), _f64(t["residual"]), options)
    # in place
    y, r = t["y"].clone(), t["residual"].clone()
    got = pdx.block_norm(y, r, stream_out=r, out=y, **options)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("tokens,hidden,top_k", tuple((t, h, (1, 3, 5, 8)[i % 4]) for i, (t, h) in enumerate(MANY_ROWS))
                         + ((593, 2048, 32), (593, 511, 32)))
@pytest.mark.parametrize("residual", (torch.bfloat16, torch.float32))
@pytest.mark.parametrize("post,pre,gate,act", (("rms", "rms", "token", "sigmoid"), ("layer", "layer", "full", "sigmoid"),
                                               ("none", "rms", "channel", "none")))
def test_many_combined_rows(pdx, tokens, hidden, top_k, residual, post, pre, gate, act):
    t = _inputs(tokens, hidden, residual, gate, seed=hidden + top_k)
    gen = torch.Generator().manual_seed(tokens)
    rows = torch.randn(tokens * top_k, hidden, generator=gen).to(torch.bfloat16).cuda()
    weights = torch.rand(tokens, top_k, generator=gen).to(torch.bfloat16).cuda()
    inverse = torch.randperm(tokens * top_k, generator=gen).to(torch.int32).cuda()
    options = dict(post=post, pre=pre, gate=t["gate"], gate_act=act, pre_weight=t["pre_weight"],
                   post_weight=t["post_weight"] if post != "none" else None)
    want = pdx.combine_block_norm(rows, weights, inverse, t["residual"], **options)
    y = np.einsum("tkh,tk->th", _f64(rows)[inverse.cpu().numpy()].reshape(tokens, top_k, hidden), _f64(weights))
    # the FP32 combine is off by top_k 2^-24 of the magnitudes of its terms, which for up to 32 terms of both
    # signs stays inside _check's 2^-17 of the row's largest sum
    _check(want, y, _f64(t["residual"]), options)
    r = t["residual"].clone()
    got = pdx.combine_block_norm(rows, weights, inverse, r, stream_out=r, **options)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_many_rows_from_an_odd_address(pdx):
    """Rows of whole vectors whose base is no multiple of 16 bytes go value by value."""
    t = _inputs(600, 1024, torch.bfloat16, "full", seed=3)
    want = pdx.block_norm(t["y"], t["residual"], post="rms", gate=t["gate"])
    _check(want, _f64(t["y"]), _f64(t["residual"]), dict(post="rms", gate=t["gate"]))
    odd = torch.empty(600 * 1024 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(600, 1024).copy_(t["y"])
    options = dict(post="rms", gate=t["gate"])
    _check(pdx.block_norm(odd, t["residual"], **options), _f64(t["y"]), _f64(t["residual"]), options)
