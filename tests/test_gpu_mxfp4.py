"""MXFP4 quantisation (bit for bit) and the grouped experts on MXFP4 weights,
against their 64-bit definitions."""
import numpy as np
import pytest
import torch

from tests import mxfp4_ref as ref

pytestmark = pytest.mark.gpu

TYPES = (torch.bfloat16, torch.float16, torch.float32)


@pytest.fixture(scope="module")
def pdx():
    import pdscope_b200
    return pdscope_b200


def _check_quantised(pdx, x):
    q = pdx.quantize_mxfp4(x)
    codes, scales = ref.quantize(x.double().cpu().numpy())
    assert np.array_equal(q.scales.cpu().numpy(), scales)
    assert np.array_equal(q.codes.cpu().numpy(), codes)
    return q


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", ((1, 32), (1, 64), (3, 96), (37, 1056), (700, 2048), (2, 5, 160), (64,)))
def test_quantize(pdx, dtype, shape):
    gen = torch.Generator().manual_seed(len(shape) * 1000 + shape[-1])
    x = torch.randn(shape, generator=gen) * torch.exp2(torch.randint(-12, 12, shape, generator=gen).float())
    _check_quantised(pdx, x.to(dtype).cuda())


@pytest.mark.parametrize("dtype", TYPES)
def test_quantize_borders(pdx, dtype):
    """Every midpoint of the grid and its neighbours at several scales, signed
    zeros, an all-zero block, subnormals and the type's largest values."""
    mids = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.5]
    block = torch.tensor([4.0] + mids + [-m for m in mids] + [0.0, -0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 6.0, -6.0, 0.24, 0.26])
    info = torch.finfo(dtype)
    rows = [block * 2.0 ** e for e in (-10, -3, 0, 5, 10)]
    rows += [torch.zeros(32), torch.full((32,), info.max), torch.full((32,), -info.tiny),
             torch.linspace(-1, 1, 32) * info.tiny, torch.linspace(0, 1, 32) * info.max]
    sub = torch.zeros(32)
    sub[3], sub[4] = info.smallest_normal * info.eps, -3 * info.smallest_normal * info.eps
    _check_quantised(pdx, torch.stack(rows + [sub]).to(dtype).cuda())


@pytest.mark.parametrize("bad", (float("inf"), float("-inf"), float("nan")))
def test_quantize_non_finite(pdx, bad):
    x = torch.randn(4, 96, generator=torch.Generator().manual_seed(5)).cuda()
    x[1, 40] = bad
    q = _check_quantised(pdx, x)
    v = pdx.dequantize_mxfp4(q, torch.float32)
    assert v[1, 32:64].isnan().all() and v.isnan().sum() == 32


def test_quantize_strided_and_unaligned(pdx):
    base = torch.randn(40, 200, generator=torch.Generator().manual_seed(9)).cuda()
    for view in (base[:, :96], base[:, 4:100], base[1::3, 3:99], base.to(torch.bfloat16)[:, 1:161]):
        _check_quantised(pdx, view)
    q = pdx.quantize_mxfp4(torch.empty(0, 64, device="cuda"))
    assert q.codes.shape == (0, 32) and pdx.dequantize_mxfp4(q).shape == (0, 64)


@pytest.mark.parametrize("dtype", TYPES)
def test_dequantize_every_code_and_scale(pdx, dtype):
    codes = torch.arange(256, dtype=torch.uint8).repeat_interleave(16).view(256, 16)
    codes = codes.roll(3, 0).cuda()      # a code pair per row, every pair once
    scales = torch.arange(256, dtype=torch.uint8).view(256, 1).cuda()
    got = pdx.dequantize_mxfp4(pdx.Mxfp4(codes, scales), dtype)
    want = torch.from_numpy(ref.dequantize(codes.cpu().numpy(), scales.cpu().numpy())).to(torch.float32).to(dtype)
    assert torch.equal(got.cpu().nan_to_num(nan=-7), want.nan_to_num(nan=-7))
    assert torch.equal(got.cpu().isnan(), want.isnan())


# ---------------------------------------------------------------------------
# Grouped experts
# ---------------------------------------------------------------------------


def _slab(pdx, experts, hidden, inter, seed, std=0.02):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    qs = [pdx.quantize_mxfp4(torch.randn(experts, r, c, device="cuda", generator=gen) * std)
          for r, c in ((inter, hidden), (inter, hidden), (hidden, inter))]
    return pdx.Mxfp4ExpertSlab.from_quantized(*qs), qs


def _weights64(qs, e):
    return [ref.dequantize(q.codes[e].cpu().numpy(), q.scales[e].cpu().numpy()) for q in qs]


def _selected(tokens, experts, k, seed, only=None):
    gen = torch.Generator().manual_seed(seed)
    score = torch.rand(tokens, experts, generator=gen)
    if only is not None:
        score[:, only] += 10
    return torch.topk(score, k, dim=1).indices.contiguous().cuda()


def _check_rows(got, x, packed, qs, experts):
    """Every expert's rows (at most 80 of each) within the derived bound."""
    offsets, tokens = packed.offsets.cpu().tolist(), packed.tokens.cpu().numpy()
    x64, got64 = x.double().cpu().numpy(), got.double().cpu().numpy()
    for e in range(experts):
        a, b = offsets[e], offsets[e + 1]
        if a == b:
            continue
        rows = np.arange(a, b)
        if len(rows) > 80:
            rows = np.unique(np.concatenate([rows[:24], rows[-24:], rows[::max(1, len(rows) // 32)]]))
        y, bound = ref.ffn_rows(x64[tokens[rows]], *_weights64(qs, e))
        err = np.abs(got64[rows] - y)
        assert (err <= bound).all(), (e, float((err / bound).max()))


SHAPES = [  # tokens, hidden, inter, experts, top_k
    (1, 32, 32, 1, 1), (1, 128, 128, 4, 2), (1, 2048, 768, 16, 8), (2, 96, 160, 3, 3), (7, 256, 128, 8, 2),
    (16, 1056, 416, 6, 4), (33, 512, 96, 5, 1), (64, 384, 256, 24, 8), (65, 2048, 768, 4, 2), (129, 640, 288, 3, 2),
    (257, 256, 128, 2, 1), (300, 128, 1024, 9, 3), (1000, 256, 256, 4, 4),
    # several tiles for every CTA or pair: narrow, middle and wide token tiles, odd numbers of 128-row blocks
    (200, 640, 640, 120, 8), (380, 384, 1152, 100, 8), (600, 256, 1280, 100, 6), (4100, 1152, 896, 4, 2),
    # as many experts as the tables hold
    (70, 128, 128, 1024, 8), (1, 8192, 64, 2, 1),
    # wide tiles whose K is cut up: in the first product, in the second
    (120, 4096, 128, 1, 1), (120, 128, 4096, 1, 1),
]


@pytest.mark.parametrize("tokens,hidden,inter,experts,top_k", SHAPES)
def test_grouped_ffn(pdx, tokens, hidden, inter, experts, top_k):
    slab, qs = _slab(pdx, experts, hidden, inter, seed=hidden + tokens)
    x = torch.randn(tokens, hidden, generator=torch.Generator().manual_seed(tokens)).to(torch.bfloat16).cuda()
    sel = _selected(tokens, experts, top_k, seed=tokens + 1)
    packed = pdx.pack(sel, torch.ones(sel.shape, dtype=torch.bfloat16, device="cuda"), experts)
    got = pdx.moe_ffn_mxfp4(x, packed, slab)
    _check_rows(got, x, packed, qs, experts)
    # the same call gives the same bits
    assert torch.equal(got, pdx.moe_ffn_mxfp4(x, packed, slab))


@pytest.mark.parametrize("std,scale", ((0.02, 1e-30), (1e4, 1e-3), (0.02, 1e4), (1e-20, 1e10)))
def test_grouped_ffn_ranges(pdx, std, scale):
    """Far from unit scale: the pieces are scaled to the row's and the block's largest value."""
    slab, qs = _slab(pdx, 4, 256, 128, seed=3, std=std)
    x = (torch.randn(20, 256, generator=torch.Generator().manual_seed(1)) * scale).to(torch.bfloat16)
    x[:, 7] *= 200          # an outlier channel
    x[3] = 0                # a row of zeros
    x = x.cuda()
    sel = _selected(20, 4, 2, seed=2)
    packed = pdx.pack(sel, torch.ones(sel.shape, dtype=torch.bfloat16, device="cuda"), 4)
    got = pdx.moe_ffn_mxfp4(x, packed, slab)
    _check_rows(got, x, packed, qs, 4)
    zero = (packed.tokens == 3).nonzero().flatten()
    assert (got[zero] == 0).all()


@pytest.mark.parametrize("tokens", (3, 40, 300))      # the three token tiles
def test_outlier_the_weights_ignore(pdx, tokens):
    """A channel 4000 times the rest whose weights are zero: what is left of the
    others' precision (2^-21 of the row's largest value each) decides."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    ws = [torch.randn(2, r, c, device="cuda", generator=gen) * 0.05 for r, c in ((128, 512), (128, 512), (512, 128))]
    ws[0][:, :, 77], ws[1][:, :, 77] = 0, 0
    qs = [pdx.quantize_mxfp4(w) for w in ws]
    slab = pdx.Mxfp4ExpertSlab.from_quantized(*qs)
    x = torch.randn(tokens, 512, device="cuda", generator=gen)
    x[:, 77] = 4000.0
    x = x.to(torch.bfloat16)
    sel = _selected(tokens, 2, 1, seed=1)
    packed = pdx.pack(sel, torch.ones(sel.shape, dtype=torch.bfloat16, device="cuda"), 2)
    got = pdx.moe_ffn_mxfp4(x, packed, slab)
    _check_rows(got, x, packed, qs, 2)
    x[:, 77] = 0
    clean = pdx.moe_ffn_mxfp4(x, packed, slab)
    # 4000 2^-21 = 2^-9 at most of values of about 1, averaged over 512: below BF16's own rounding
    assert (got.double() - clean.double()).norm() <= 2.0 ** -8 * clean.double().norm()


@pytest.mark.parametrize("bad", (float("inf"), float("nan")))
def test_non_finite_rows_stay_in_their_rows(pdx, bad):
    slab, _ = _slab(pdx, 4, 256, 128, seed=3)
    x = torch.randn(40, 256, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    sel = _selected(40, 4, 2, seed=2)
    packed = pdx.pack(sel, torch.ones(sel.shape, dtype=torch.bfloat16, device="cuda"), 4)
    clean = pdx.moe_ffn_mxfp4(x, packed, slab)
    x[5, 100] = bad
    got = pdx.moe_ffn_mxfp4(x, packed, slab)
    hit = packed.tokens == 5
    assert (~got[hit].isfinite()).all()
    assert torch.equal(got[~hit], clean[~hit])


def test_nan_weight_block_reaches_its_outputs(pdx):
    """A NaN scale in one expert's gate row makes that expert's rows NaN, no other's."""
    slab, qs = _slab(pdx, 4, 256, 128, seed=3)
    qs[0].scales[2, 17, 3] = 255
    slab.store(0, *qs)
    x = torch.randn(24, 256, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    sel = _selected(24, 4, 2, seed=2)
    packed = pdx.pack(sel, torch.ones(sel.shape, dtype=torch.bfloat16, device="cuda"), 4)
    got = pdx.moe_ffn_mxfp4(x, packed, slab)
    a, b = packed.offsets[2].item(), packed.offsets[3].item()
    assert got[a:b].isnan().all()
    assert got[:a].isfinite().all() and got[b:].isfinite().all()


def test_slots_empty_experts_and_spare_rows(pdx):
    """Experts in other slots, experts without rows, and rows of no active
    expert left as they were."""
    experts, hidden, inter = 6, 256, 128
    slab, qs = _slab(pdx, experts, hidden, inter, seed=11)
    order = torch.tensor([4, 2, 0, 5, 1, 3], dtype=torch.int32, device="cuda")
    moved = pdx.Mxfp4ExpertSlab(experts, hidden, inter, "cuda", slot_of_expert=order)
    for e in range(experts):
        moved.store(int(order[e]), *(pdx.Mxfp4(q.codes[e:e + 1], q.scales[e:e + 1]) for q in qs))
    x = torch.randn(50, hidden, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    sel = _selected(50, experts, 2, seed=3, only=[1, 4])       # four experts have no rows
    packed = pdx.pack(sel, torch.ones(sel.shape, dtype=torch.bfloat16, device="cuda"), experts)
    got = pdx.moe_ffn_mxfp4(x, packed, moved)
    assert torch.equal(got, pdx.moe_ffn_mxfp4(x, packed, slab))
    _check_rows(got, x, packed, qs, experts)
    # only expert 4 active: expert 1's rows stay
    packed.active[0], packed.active[1] = 1, 4
    out = torch.full_like(got, 7.0)
    pdx.moe_ffn_mxfp4(x, packed, slab, out=out)
    a, b = packed.offsets[4].item(), packed.offsets[5].item()
    assert torch.equal(out[a:b], got[a:b])
    assert (out[:a] == 7).all() and (out[b:] == 7).all()


@pytest.mark.parametrize("tokens", (2, 60, 400))      # the three token tiles
def test_active_list_may_name_empty_experts(pdx, tokens):
    slab, qs = _slab(pdx, 6, 256, 128, seed=12)
    x = torch.randn(tokens, 256, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    sel = _selected(tokens, 6, 2, seed=3, only=[1, 4])
    packed = pdx.pack(sel, torch.ones(sel.shape, dtype=torch.bfloat16, device="cuda"), 6)
    want = pdx.moe_ffn_mxfp4(x, packed, slab)
    _check_rows(want, x, packed, qs, 6)
    n = min(6, packed.tokens.shape[0])                   # every expert, the empty ones too
    packed.active[:n + 1] = torch.tensor([n, 0, 1, 2, 3, 4, 5][:n + 1], dtype=torch.int32)
    if n == 6:
        assert torch.equal(pdx.moe_ffn_mxfp4(x, packed, slab), want)


@pytest.mark.parametrize("tokens", (1, 60, 400))
def test_inputs_written_just_before_the_call(pdx, tokens):
    """Weights, routing and activations written on the same stream right before:
    the launches that start early must not read what was there."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    sets = []
    for i in range(2):
        slab, qs = _slab(pdx, 8, 512, 256, seed=20 + i)
        x = torch.randn(tokens, 512, device="cuda", generator=gen).to(torch.bfloat16)
        sel = _selected(tokens, 8, 2, seed=30 + i)
        packed = pdx.pack(sel, torch.ones(sel.shape, dtype=torch.bfloat16, device="cuda"), 8)
        sets.append((slab, x, sel, pdx.moe_ffn_mxfp4(x, packed, slab)))
    slab, x = pdx.Mxfp4ExpertSlab(8, 512, 256, "cuda"), torch.empty_like(sets[0][1])
    sel, ones = torch.empty_like(sets[0][2]), torch.ones(sets[0][2].shape, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    got = []
    for i in range(12):
        src = sets[i % 2]
        sel.copy_(src[2])
        x.copy_(src[1])
        slab.scales.copy_(src[0].scales)
        slab.codes.copy_(src[0].codes)
        got.append(pdx.moe_ffn_mxfp4(x, pdx.pack(sel, ones, 8), slab))
    for i, y in enumerate(got):
        assert torch.equal(y, sets[i % 2][3]), i


def test_bad_slot_and_bad_token_are_reported(pdx):
    from pdscope_b200 import runtime
    slab, qs = _slab(pdx, 4, 256, 128, seed=11)
    wrong = pdx.Mxfp4ExpertSlab(4, 256, 128, "cuda",
                                slot_of_expert=torch.tensor([0, 9, 2, 3], dtype=torch.int32, device="cuda"))
    wrong.store(0, *qs)
    x = torch.randn(8, 256, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    sel = _selected(8, 4, 2, seed=3, only=[1])
    packed = pdx.pack(sel, torch.ones(sel.shape, dtype=torch.bfloat16, device="cuda"), 4)
    pdx.moe_ffn_mxfp4(x, packed, wrong)
    with pytest.raises(ValueError, match="slot"):
        runtime.raise_device_error()
    packed.tokens[0] = 8
    pdx.moe_ffn_mxfp4(x, packed, slab)
    with pytest.raises(ValueError, match="expert ID"):
        runtime.raise_device_error()
    runtime.raise_device_error()


def test_streams_and_graphs_at_once(pdx):
    """Calls on several streams at once and captured graphs replayed in turn
    give what single calls give."""
    cases = []
    for tokens, seed in ((48, 1), (3, 2), (900, 3)):   # the three token tiles
        slab, _ = _slab(pdx, 8, 512, 256, seed=seed)
        x = torch.randn(tokens, 512, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()
        sel = _selected(tokens, 8, 4, seed=seed)
        packed = pdx.pack(sel, torch.ones(sel.shape, dtype=torch.bfloat16, device="cuda"), 8)
        cases.append((x, packed, slab, pdx.moe_ffn_mxfp4(x, packed, slab)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    outs = []
    for _ in range(10):
        for stream, (x, packed, slab, _) in zip(streams, cases):
            with torch.cuda.stream(stream):
                outs.append(pdx.moe_ffn_mxfp4(x, packed, slab))
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        assert torch.equal(out, cases[i % len(cases)][3])
    graphs = []
    for x, packed, slab, want in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = pdx.moe_ffn_mxfp4(x, packed, slab)
        graphs.append((g, out, want))
    for _ in range(3):
        for g, out, _ in graphs:
            out.zero_()
            g.replay()
        torch.cuda.synchronize()
        for _, out, want in graphs:
            assert torch.equal(out, want)


def test_slab_round_trip(pdx):
    """from_slab, from_tensors, load and expert_tensors agree; a quantised slab
    quantises to itself."""
    slab = pdx.ExpertSlab.allocate(3, 160, 96, "cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    a = pdx.Mxfp4ExpertSlab.from_slab(slab)
    b = pdx.Mxfp4ExpertSlab.from_tensors([slab.expert_tensors(s) for s in range(3)])
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    for s in range(3):
        for name, t in a.expert_tensors(s).items():
            codes, scales = ref.quantize(slab.expert_tensors(s)[name].double().cpu().numpy())
            assert np.array_equal(t.double().cpu().numpy(), ref.dequantize(codes, scales))
    again = pdx.Mxfp4ExpertSlab.from_tensors([a.expert_tensors(s) for s in range(3)])
    for s in range(3):
        for name, t in a.expert_tensors(s).items():
            assert torch.equal(again.expert_tensors(s)[name], t)


@pytest.mark.parametrize("tokens", (1, 5, 70))
def test_layer_is_its_parts(pdx, tokens):
    """ResidentMoELayer on an MXFP4 slab: route, pack, moe_ffn_mxfp4, combine."""
    experts, hidden, inter = 16, 512, 256
    slab, _ = _slab(pdx, experts, hidden, inter, seed=tokens)
    gen = torch.Generator().manual_seed(tokens)
    gate = (torch.randn(experts, hidden, generator=gen) * 0.05).to(torch.bfloat16).cuda()
    x = torch.randn(tokens, hidden, generator=gen).to(torch.bfloat16).cuda()
    layer = pdx.ResidentMoELayer(gate, slab, top_k=4)
    out = layer.forward(x)
    r = pdx.route(x, gate, 4, True)
    packed = pdx.pack(r.selected, r.weights, experts)
    rows = pdx.moe_ffn_mxfp4(x, packed, slab)
    assert torch.equal(out.selected, r.selected)
    assert torch.equal(out.out, pdx.combine(rows, r.weights, packed.inverse))
    assert torch.equal(out.counts, packed.counts)


def test_runtime_forward_on_mxfp4(pdx):
    experts, hidden, inter = 8, 256, 128
    slab, _ = _slab(pdx, experts, hidden, inter, seed=1)
    gen = torch.Generator().manual_seed(3)
    gate = (torch.randn(experts, hidden, generator=gen) * 0.05).to(torch.bfloat16).cuda()
    x = torch.randn(12, hidden, generator=gen).to(torch.bfloat16).cuda()
    rt = pdx.PDScopeCudaRuntime({0: slab}, top_k=2)
    out, routing, row = rt.forward(x, gate, layer=0, step=0, top_k=2)
    assert torch.equal(out, pdx.ResidentMoELayer(gate, slab, top_k=2).forward(x).out)
    assert row["counters"]["gpu_completed_experts"] == len(row["token_counts"])


@pytest.mark.parametrize("tokens,hidden,inter,experts,top_k", ((1, 2048, 768, 16, 8), (3, 1024, 1024, 4, 2),
                                                               (120, 4096, 128, 1, 1), (120, 128, 4096, 1, 1)))
def test_joined_parts_repeat(pdx, tokens, hidden, inter, experts, top_k):
    """Tiles whose K is cut up between CTAs, back to back: every join reads the
    parts of its own call, whichever CTA comes last."""
    slab, qs = _slab(pdx, experts, hidden, inter, seed=21)
    sets = []
    for i in range(2):
        x = torch.randn(tokens, hidden, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16).cuda()
        sel = _selected(tokens, experts, top_k, seed=i)
        packed = pdx.pack(sel, torch.ones(sel.shape, dtype=torch.bfloat16, device="cuda"), experts)
        want = pdx.moe_ffn_mxfp4(x, packed, slab)
        _check_rows(want, x, packed, qs, experts)
        sets.append((x, packed, want))
    outs = [pdx.moe_ffn_mxfp4(*sets[i % 2][:2], slab) for i in range(200)]
    for i, out in enumerate(outs):
        assert torch.equal(out, sets[i % 2][2]), i


@pytest.mark.parametrize("tokens,experts", ((1, 6), (2, 6), (8, 6), (2, 1024), (40, 6), (400, 6)))
def test_active_list_longer_than_the_rows(pdx, tokens, experts):
    """Every expert listed, the empty ones first: those with rows still run."""
    slab, qs = _slab(pdx, experts, 128, 128, seed=12)
    x = torch.randn(tokens, 128, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    sel = _selected(tokens, experts, 2, seed=3, only=[1, 4])
    packed = pdx.pack(sel, torch.ones(sel.shape, dtype=torch.bfloat16, device="cuda"), experts)
    want = pdx.moe_ffn_mxfp4(x, packed, slab)
    _check_rows(want, x, packed, qs, experts)
    ids = torch.arange(experts - 1, -1, -1, dtype=torch.int32)
    packed.active.copy_(torch.cat([torch.tensor([experts], dtype=torch.int32), ids]))
    out = torch.full_like(want, 7.0)
    assert torch.equal(pdx.moe_ffn_mxfp4(x, packed, slab, out=out), want)


@pytest.mark.parametrize("tokens", (2, 60, 400))      # the three token tiles
@pytest.mark.parametrize("active", ((2, 1, 1), (2, 1, 99), (2, 1, 6), (1, -1), (7, 0, 1, 2, 3, 4, 5), (6, 1, 1, 1, 1, 1, 1)))
def test_bad_active_lists_are_reported(pdx, tokens, active):
    """Ids out of range, more entries than experts, an expert named again and
    again: an error word, and nothing outside the rows is touched."""
    from pdscope_b200 import runtime
    slab, _ = _slab(pdx, 6, 128, 128, seed=12)
    x = torch.randn(tokens, 128, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    sel = _selected(tokens, 6, 2, seed=3, only=[1, 4])
    packed = pdx.pack(sel, torch.ones(sel.shape, dtype=torch.bfloat16, device="cuda"), 6)
    want = pdx.moe_ffn_mxfp4(x, packed, slab)
    good = packed.active.clone()
    packed.active[:len(active)] = torch.tensor(active, dtype=torch.int32)
    guard = torch.full((2 * tokens + 2, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    pdx.moe_ffn_mxfp4(x, packed, slab, out=guard[1:-1])
    assert (guard[0] == 7).all() and (guard[-1] == 7).all()
    if active == (2, 1, 1):                               # the same rows twice, the same values
        a, b = packed.offsets[1].item(), packed.offsets[2].item()
        assert torch.equal(guard[1 + a:1 + b], want[a:b])
    else:
        with pytest.raises(ValueError, match="expert ID"):
            runtime.raise_device_error()
    runtime.raise_device_error()
    packed.active.copy_(good)
    assert torch.equal(pdx.moe_ffn_mxfp4(x, packed, slab), want)


@pytest.mark.parametrize("tokens", (2, 400))
def test_bad_offsets_are_reported(pdx, tokens):
    from pdscope_b200 import runtime
    slab, _ = _slab(pdx, 6, 128, 128, seed=12)
    x = torch.randn(tokens, 128, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).cuda()
    sel = _selected(tokens, 6, 2, seed=3, only=[1, 4])
    packed = pdx.pack(sel, torch.ones(sel.shape, dtype=torch.bfloat16, device="cuda"), 6)
    good = packed.offsets.clone()
    for bad in ((5, 2 * tokens + 1), (1, -1), (2, -5)):       # past the rows, before them, falling
        packed.offsets.copy_(good)
        packed.offsets[bad[0]] = bad[1]
        guard = torch.full((2 * tokens + 2, 128), 7.0, dtype=torch.bfloat16, device="cuda")
        pdx.moe_ffn_mxfp4(x, packed, slab, out=guard[1:-1])
        assert (guard[0] == 7).all() and (guard[-1] == 7).all()
        with pytest.raises(ValueError, match="expert ID"):
            runtime.raise_device_error()


# more than 592 packed rows of more than 2048 channels: one warp a row, rows longer than it holds at once
LONG_ROWS = ((80, 4096, 64, 120, 8), (100, 2080, 96, 100, 7), (200, 2176, 96, 40, 8), (700, 4128, 96, 3, 1),
             (640, 8192, 64, 2, 1))


@pytest.mark.parametrize("tokens,hidden,inter,experts,top_k", LONG_ROWS)
def test_many_long_rows(pdx, tokens, hidden, inter, experts, top_k):
    slab, qs = _slab(pdx, experts, hidden, inter, seed=hidden + tokens)
    x = torch.randn(tokens, hidden, generator=torch.Generator().manual_seed(tokens)).to(torch.bfloat16)
    x[:, hidden - 3] *= 50        # in the last values of a row
    x = x.cuda()
    sel = _selected(tokens, experts, top_k, seed=tokens + 1)
    packed = pdx.pack(sel, torch.ones(sel.shape, dtype=torch.bfloat16, device="cuda"), experts)
    got = pdx.moe_ffn_mxfp4(x, packed, slab)
    _check_rows(got, x, packed, qs, experts)


@pytest.mark.parametrize("tokens", (3, 40, 300))      # the three token tiles
def test_far_outlier_the_weights_ignore(pdx, tokens):
    """A channel 2^15 times the rest whose weights are zero takes bits only from
    the 31 values that share its block."""
    gen = torch.Generator(device="cuda").manual_seed(7)
    ws = [torch.randn(2, r, c, device="cuda", generator=gen) * 0.02 for r, c in ((128, 2048), (128, 2048), (2048, 128))]
    ws[0][:, :, 77], ws[1][:, :, 77] = 0, 0
    qs = [pdx.quantize_mxfp4(w) for w in ws]
    slab = pdx.Mxfp4ExpertSlab.from_quantized(*qs)
    x = torch.randn(tokens, 2048, device="cuda", generator=gen)
    x[:, 77] = 2.0 ** 15
    x = x.to(torch.bfloat16)
    sel = _selected(tokens, 2, 1, seed=1)
    packed = pdx.pack(sel, torch.ones(sel.shape, dtype=torch.bfloat16, device="cuda"), 2)
    got = pdx.moe_ffn_mxfp4(x, packed, slab).double().cpu().numpy()
    offsets, order, x64 = packed.offsets.tolist(), packed.tokens.cpu().numpy(), x.double().cpu().numpy()
    y = np.concatenate([ref.ffn_rows(x64[order[offsets[e]:offsets[e + 1]]], *_weights64(qs, e))[0] for e in range(2)])
    # 31 of 2048 values off by 2^-21 2^15 = 2^-6 at most: 2^-6 sqrt(31/2048) = 1.9e-3 of gate and of up, 3.8e-3 of h;
    # the roundings of h and y 2^-8 each: in quadrature 6.7e-3 < 2^-7
    assert np.linalg.norm(got - y) <= 2.0 ** -7 * np.linalg.norm(y)


@pytest.mark.parametrize("tokens,hidden", ((1, 96), (3, 1024), (40, 1056), (300, 2080)))
def test_blocks_of_far_apart_sizes(pdx, tokens, hidden):
    """Blocks of 32 channels from 2^-30 to 2^30 times the first, weights the other
    way round: every block counts alike, and a power of two changes no bit of a product."""
    gen = torch.Generator(device="cuda").manual_seed(9)
    ws = [torch.randn(3, r, c, device="cuda", generator=gen) * 0.05 for r, c in ((160, hidden), (160, hidden), (hidden, 160))]
    x = torch.randn(tokens, hidden, device="cuda", generator=gen).to(torch.bfloat16)
    sel = _selected(tokens, 3, 1, seed=1)
    packed = pdx.pack(sel, torch.ones(sel.shape, dtype=torch.bfloat16, device="cuda"), 3)
    power = torch.exp2(((torch.arange(hidden, device="cuda") // 32 * 17) % 61 - 30).float())
    qs = [pdx.quantize_mxfp4(ws[0] / power), pdx.quantize_mxfp4(ws[1] / power), pdx.quantize_mxfp4(ws[2])]
    slab = pdx.Mxfp4ExpertSlab.from_quantized(*qs)
    got = pdx.moe_ffn_mxfp4((x.float() * power).to(torch.bfloat16), packed, slab)
    offsets, order = packed.offsets.tolist(), packed.tokens.cpu().numpy()
    x64, wide = x.double().cpu().numpy(), power.double().cpu().numpy()
    for e in range(3):
        rows = slice(offsets[e], offsets[e + 1])
        if rows.start == rows.stop:
            continue
        g, u, d = _weights64(qs, e)
        y, bound = ref.ffn_rows(x64[order[rows]], g * wide, u * wide, d)     # as if every block were of the first's size
        assert (np.abs(got[rows].double().cpu().numpy() - y) <= bound).all()


# the split of x with one, two and four blocks of 512 columns in flight, narrow and wide token tiles
SPLITS = ((900, 128, 64, 120, 8), (900, 1024, 64, 60, 8), (4000, 640, 64, 9, 2), (3600, 1056, 64, 120, 2),
          (1000, 4096, 32, 130, 7), (1300, 2080, 32, 5, 3))


@pytest.mark.parametrize("tokens,hidden,inter,experts,top_k", SPLITS)
def test_split_forms(pdx, tokens, hidden, inter, experts, top_k):
    slab, qs = _slab(pdx, experts, hidden, inter, seed=hidden + tokens)
    gen = torch.Generator().manual_seed(tokens)
    x = torch.randn(tokens, hidden, generator=gen) * torch.exp2(torch.randint(-8, 8, (tokens, 1), generator=gen).float())
    x[:, ::97] *= 300
    x = x.to(torch.bfloat16).cuda()
    sel = _selected(tokens, experts, top_k, seed=tokens + 1)
    packed = pdx.pack(sel, torch.ones(sel.shape, dtype=torch.bfloat16, device="cuda"), experts)
    got = pdx.moe_ffn_mxfp4(x, packed, slab)
    _check_rows(got, x, packed, qs, experts)
    assert torch.equal(got, pdx.moe_ffn_mxfp4(x, packed, slab))
