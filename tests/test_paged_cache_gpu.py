"""GPU tests of the paged cache: each operator against a plain implementation (64 bits, or whole numbers), where it can go wrong;
then a run of them together, as a server uses them."""
import ctypes
import math

import pytest
import torch

import triton_flashattn_b200 as fa
from triton_flashattn_b200 import _cabi

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16
INF = float("inf")


# ---------------------------------------------------------------------------------- attention
def attend_ref(q, k_cache, v_cache, table, lens, bias=None, scale=None):
    """(result, tolerance) in 64 bits, from the definition, sequence by sequence.

    The tolerance of an element, with u = eps / 2 the rounding of the 16-bit type and w the normalised weights:
      * the result is rounded once: u |o|
      * a score is a sum of D exact products in fp32, times the scale, plus the bias, times log2 e: its error is at most
        ds = (D + 4) 2^-24 scale sum|q k| + 2^-22 (|s| + |max|); the exponential adds 2^-21 relative; numerator and sum have it: twice
      * a weight enters the product as two 16-bit terms: u^2 relative (fp16: not below 2^-25 of the largest weight, an absolute step)
      * sums over n keys in fp32, in numerator and sum, and over the joints: 2 (n + 64) 2^-24 relative
    each relative one times sum w |v|."""
    B, H, D = q.shape
    pages, page, Hkv, _ = k_cache.shape
    scale = D ** -0.5 if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    out, tol = torch.zeros(B, H, D, dtype=torch.float64), torch.zeros(B, H, D, dtype=torch.float64)
    table, lens = table.cpu().long(), lens.cpu().tolist()
    for b in range(B):
        n = min(max(lens[b], 0), table.shape[1] * page)
        at = torch.arange(n)
        ids = table[b, at // page]
        at = at[(ids >= 0) & (ids < pages)]
        if len(at) == 0:
            continue
        ids, rows = table[b, at // page].to(q.device), (at % page).to(q.device)
        k, v = k_cache[ids, rows].double().cpu(), v_cache[ids, rows].double().cpu()
        for h in range(H):
            kh, vh, qh = k[:, h // (H // Hkv)], v[:, h // (H // Hkv)], q[b, h].double().cpu()
            s, size = kh @ qh * scale, (kh.abs() @ qh.abs()) * abs(scale)
            if bias is not None:
                x = bias[b, h].cpu()[at]
                s = torch.where(x, s, -INF) if bias.dtype == torch.bool else s + x.double()
            part = s != -INF
            if not part.any():
                continue
            s, size, vh = s[part], size[part], vh[part]
            w = torch.exp(s - s.max())
            total = w.sum()
            w = w / total
            out[b, h] = w @ vh
            # (weights that vanish do so with any error of theirs)
            near = (s - s.max()) > -60
            ds = (D + 4) * 2.0 ** -24 * size[near].max() + 2.0 ** -22 * (s[near].abs().max() + s.max().abs())
            rel = 2 * (ds + 2.0 ** -21) + u * u + 2 * (len(s) + 64) * 2.0 ** -24
            tol[b, h] = u * out[b, h].abs() + rel * (w @ vh.abs())
            if q.dtype == HF:
                tol[b, h] += len(s) * 2.0 ** -25 / total * vh.abs().max() + 2.0 ** -25
    return out, tol


def make_cache(lens, page, Hkv, D, dtype, seed, width=None, stale=float("nan")):
    """(k_cache, v_cache, block_table, seq_lens): pages anywhere, whatever no sequence holds filled with `stale`."""
    g = torch.Generator().manual_seed(seed)
    held = [-(-max(n, 0) // page) for n in lens]
    width = max(max(held), 1) if width is None else width
    pages = sum(held) + 3
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(lens), width), -7, dtype=torch.int32)
    k, v = (torch.full((pages, page, Hkv, D), stale) for _ in range(2))
    at = 0
    for b, n in enumerate(lens):
        table[b, :held[b]] = order[at:at + held[b]].int()
        at += held[b]
        pos = torch.arange(max(n, 0))
        ids, rows = table[b].long()[pos // page], pos % page
        k[ids, rows] = torch.randn(max(n, 0), Hkv, D, generator=g)
        v[ids, rows] = torch.randn(max(n, 0), Hkv, D, generator=g)
    return (k.to(dtype).cuda(), v.to(dtype).cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32, device="cuda"))


def make_q(B, H, D, dtype, seed):
    return torch.randn(B, H, D, generator=torch.Generator().manual_seed(seed + 1000)).to(dtype).cuda()


def check(got, q, kc, vc, table, lens, bias=None, scale=None):
    ref, tol = attend_ref(q, kc, vc, table, lens, bias, scale)
    got = got.double().cpu()
    off = (got - ref).abs()
    assert torch.isfinite(got).all()
    worst = (off / tol.clamp(min=1e-30))[off > 0].max().item() if (off > 0).any() else 0.0
    assert (off <= tol).all(), f"off by {off.max().item():.3e}, {worst:.2f} of the tolerance"


# (lens, page, Hkv, group, D, dtype)
SHAPES = [
    ([1], 16, 1, 1, 64, BF),
    ([17], 16, 8, 4, 128, BF),
    ([0, 1, 15, 16, 17, 0], 16, 2, 3, 64, HF),
    ([63, 64, 65, 127, 128, 129], 64, 2, 8, 128, BF),
    ([1000, 3, 257, 0], 16, 3, 5, 128, HF),
    ([333], 1, 2, 2, 32, BF),
    ([100, 77], 7, 2, 7, 128, BF),
    ([130, 55], 24, 1, 16, 256, BF),
    ([400, 1, 31], 128, 4, 1, 256, HF),
    ([90, 2100], 48, 1, 9, 64, HF),
    ([45, 300], 20, 2, 12, 128, BF),
    ([513, 260], 16, 1, 32, 128, HF),
    ([70, 500], 16, 1, 41, 64, BF),
    ([64, 99], 16, 2, 4, 16, BF),
    ([5000], 1000, 1, 4, 128, BF),
    ([4097, 9], 16, 1, 1, 16, HF),
    (list(range(0, 60)), 8, 2, 2, 64, BF),
]


@pytest.mark.parametrize("lens,page,Hkv,group,D,dtype", SHAPES)
def test_attention_against_64_bits(lens, page, Hkv, group, D, dtype, device_ok):
    """Lengths from none to long, odd pages, every head dimension, groups of any size; what the sequences do not hold is NaN."""
    kc, vc, table, n = make_cache(lens, page, Hkv, D, dtype, 1)
    q = make_q(len(lens), Hkv * group, D, dtype, 1)
    check(fa.paged_attention_fn(q, kc, vc, table, n), q, kc, vc, table, n)
    check(fa.paged_attention_fn(q, kc, vc, table, n, None, -0.3), q, kc, vc, table, n, None, -0.3)


@pytest.mark.parametrize("kind", ["same", "f32", "f64", "table", "row", "strided"])
@pytest.mark.parametrize("lens,page,Hkv,group,D,dtype", [([100, 1, 777, 0], 16, 2, 4, 128, BF), ([130, 55], 24, 1, 10, 64, HF),
                                                         ([300, 20], 32, 2, 2, 256, BF)])
def test_attention_with_a_bias(lens, page, Hkv, group, D, dtype, kind, device_ok):
    kc, vc, table, n = make_cache(lens, page, Hkv, D, dtype, 2)
    B, H, N = len(lens), Hkv * group, table.shape[1] * page
    q = make_q(B, H, D, dtype, 2)
    g = torch.Generator().manual_seed(5)
    x = 2 * torch.randn(B, H, N, generator=g)
    bias = {"same": lambda: x.to(dtype).cuda(), "f32": lambda: x.cuda(), "f64": lambda: x.double().float().double().cuda(),
            "table": lambda: x[:1].cuda().expand(B, H, N), "row": lambda: x[:, :1].to(dtype).cuda().expand(B, H, N),
            "strided": lambda: x.to(dtype).cuda().transpose(1, 2).contiguous().transpose(1, 2)}[kind]()
    check(fa.paged_attention_fn(q, kc, vc, table, n, bias), q, kc, vc, table, n, bias)


@pytest.mark.parametrize("lens,page,Hkv,group,D,dtype", [([100, 1, 777, 0], 16, 2, 4, 128, BF), ([130, 55], 24, 1, 10, 64, HF),
                                                         ([300, 20], 32, 2, 2, 256, BF), ([90, 400], 5, 2, 3, 32, HF),
                                                         ([40, 210], 8, 1, 20, 128, BF), ([75, 130], 16, 1, 30, 64, HF)])
@pytest.mark.parametrize("form", ["bool", "inf", "lowest"])
def test_masks_and_what_hides_behind_them(lens, page, Hkv, group, D, dtype, form, device_ok):
    """Each head leaves out keys of its own, one head all of them, one head all but one; behind keys that every head leaves
    out lie infinities and NaN, and where one head alone looks at an infinite value the others do not see it."""
    kc, vc, table, n = make_cache(lens, page, Hkv, D, dtype, 3)
    B, H, N = len(lens), Hkv * group, table.shape[1] * page
    q = make_q(B, H, D, dtype, 3)
    g = torch.Generator().manual_seed(6)
    keep = torch.rand(B, H, N, generator=g) < 0.7
    keep[:, 1] = False
    keep[:, 0] = False
    keep[:, 0, 0] = True
    hidden = torch.rand(N, generator=g) < 0.2
    hidden[0] = False
    keep[:, :, hidden] = False
    keep, hidden = keep.cuda(), hidden.cuda()
    bias = keep if form == "bool" else torch.where(keep, 0.0, -INF if form == "inf" else torch.finfo(dtype).min).to(dtype)
    check(fa.paged_attention_fn(q, kc, vc, table, n, bias), q, kc, vc, table, n, bias)
    if form == "lowest":  # added, and no mask: a row of nothing else is the mean of its values
        return
    clean = fa.paged_attention_fn(q, kc, vc, table, n, bias)
    for b, length in enumerate(lens):
        pos = hidden[:length].nonzero()[:, 0]
        for i, at in enumerate(pos.tolist()):
            page_id = table[b, at // page]
            if form == "bool":
                kc[page_id, at % page] = (INF, -INF, float("nan"))[i % 3]
            vc[page_id, at % page] = (float("nan"), INF, -INF)[i % 3]
    assert torch.equal(fa.paged_attention_fn(q, kc, vc, table, n, bias), clean)
    # one head alone sees the first key of all
    alone = bias.clone()
    alone[:, :, 0] = False if form == "bool" else -INF
    alone[:, 0, 0] = True if form == "bool" else 0.0
    others = fa.paged_attention_fn(q, kc, vc, table, n, alone)
    for b, length in enumerate(lens):
        if length:
            vc[table[b, 0], 0] = INF
    seen = fa.paged_attention_fn(q, kc, vc, table, n, alone)
    assert torch.equal(seen[:, 1:], others[:, 1:])
    for b, length in enumerate(lens):
        if length:
            assert (seen[b, 0] == INF).all()


def test_a_bias_of_the_lowest_value_everywhere_leaves_the_mean(device_ok):
    kc, vc, table, n = make_cache([40, 133], 16, 1, 64, BF, 4)
    q = make_q(2, 4, 64, BF, 4)
    for dtype in (BF, torch.float32):
        bias = torch.full((2, 4, table.shape[1] * 16), torch.finfo(dtype).min, dtype=dtype, device="cuda")
        out = fa.paged_attention_fn(q, kc, vc, table, n, bias)
        for b, length in enumerate((40, 133)):
            pos = torch.arange(length, device="cuda")
            v = vc[table[b].long()[pos // 16], pos % 16, 0].double()
            # equal scores: equal weights, whose sums in fp32 are off by 2 n 2^-24 of sum w |v|
            tol = 2.0 ** -8 * v.mean(0).abs() + (2 * (length + 64) * 2.0 ** -24 + 2.0 ** -16) * v.abs().mean(0)
            assert ((out[b].double() - v.mean(0)).abs() <= tol).all()


def test_scores_that_are_not_finite(device_ok):
    """As the formula has it: a NaN score that takes part makes its row NaN, and so does one of +inf; other rows do not care."""
    kc, vc, table, n = make_cache([50, 50, 50], 16, 1, 64, BF, 5)
    q = make_q(3, 3, 64, BF, 5)
    bias = torch.zeros(3, 3, table.shape[1] * 16, device="cuda")
    clean = fa.paged_attention_fn(q, kc, vc, table, n, bias)
    bias[0, 0, 17], bias[1, 2, 49] = float("nan"), INF
    bias[2, 1, :] = -INF
    bias[2, 1, 3] = float("nan")
    got = fa.paged_attention_fn(q, kc, vc, table, n, bias)
    bad = [(0, 0), (1, 2), (2, 1)]
    for b in range(3):
        for h in range(3):
            assert got[b, h].isnan().all() if (b, h) in bad else torch.equal(got[b, h], clean[b, h])


def test_scores_that_jump(device_ok):
    """Scores that rise and fall by thousands along the keys: the running maximum moves in every stretch, and back."""
    kc, vc, table, n = make_cache([700, 701], 16, 2, 128, BF, 6)
    q = make_q(2, 8, 128, BF, 6)
    pos = torch.arange(table.shape[1] * 16, device="cuda").float()
    for bias in (pos * 13.7, -pos * 13.7, 3000 * torch.sin(pos), (pos == 699) * 1e30, (pos == 0) * 1e4):
        bias = bias.expand(2, 8, -1)
        check(fa.paged_attention_fn(q, kc, vc, table, n, bias), q, kc, vc, table, n, bias)


def test_lengths_and_pages_that_are_wrong(device_ok):
    """Lengths below zero and beyond the table are cut; keys on pages that the cache does not have take no part."""
    kc, vc, table, n = make_cache([64, 64, 64, 40, 64], 16, 2, 64, BF, 7)
    q = make_q(5, 4, 64, BF, 7)
    n = torch.tensor([-5, 1000, -2 ** 31, 2 ** 31 - 1, 64], dtype=torch.int32, device="cuda")
    table[1, 2], table[4, 0], table[4, 3] = -1, kc.shape[0], -2 ** 31
    table[3, 2:] = 2 ** 31 - 1
    got = fa.paged_attention_fn(q, kc, vc, table, n)
    check(got, q, kc, vc, table, n)
    assert not got[0].any() and not got[2].any()
    table[:] = -1
    assert not fa.paged_attention_fn(q, kc, vc, table, n).any()


@pytest.mark.parametrize("page", [8, 20, 1])
@pytest.mark.parametrize("D", [32, 128])
def test_wrong_pages_of_other_sizes(page, D, device_ok):
    """The same for pages that other copies bring: sequences without a key, pages that are not there first, last and between."""
    kc, vc, table, n = make_cache([64, 64, 0, 41, 64], page, 2, D, HF, 7, width=80)
    q = make_q(5, 6, D, HF, 7)
    n[2] = -3
    table[0, 0], table[1, 1], table[1, 2] = -1, kc.shape[0], 2 ** 31 - 1
    table[3, (41 - 1) // page] = -2 ** 31
    table[4] = -1
    got = fa.paged_attention_fn(q, kc, vc, table, n)
    check(got, q, kc, vc, table, n)
    assert not got[2].any() and not got[4].any()


@pytest.mark.parametrize("layout", ["heads_first", "layer", "padded", "token_first"])
def test_cache_layouts(layout, device_ok):
    lens, page, Hkv, D = [100, 300, 5], 16, 2, 64
    kc, vc, table, n = make_cache(lens, page, Hkv, D, HF, 8)
    wide = torch.randn(3, 4 * 3, 2 * D, generator=torch.Generator().manual_seed(9)).to(HF).cuda()
    q = wide[:, ::3, :D]  # heads and sequences apart
    table = torch.cat([table, table], 1)[:, :table.shape[1]]
    n = torch.stack([n, n], 1)[:, 0]
    want = fa.paged_attention_fn(q.contiguous(), kc, vc, table.contiguous(), n.contiguous())

    def laid(t):
        if layout == "heads_first":
            return t.transpose(1, 2).contiguous().transpose(1, 2)
        if layout == "layer":
            return torch.stack([t, t * 2], 1)[:, 0]
        if layout == "token_first":
            return t.transpose(0, 1).contiguous().transpose(0, 1)
        big = torch.full((t.shape[0], page + 1, Hkv + 1, D + 8), float("nan"), dtype=HF, device="cuda")
        big[:, :page, :Hkv, :D] = t
        return big[:, :page, :Hkv, :D]

    k2, v2 = laid(kc), laid(vc)
    assert not k2.is_contiguous()
    assert torch.equal(fa.paged_attention_fn(q, k2, v2, table, n), want)
    assert torch.equal(fa.paged_attention_fn(q, k2, vc, table.t().contiguous().t(), n), want)
    odd = torch.randn(3 * 4 * D + 1, device="cuda").to(HF)[1:].view(3, 4, D)  # not at a multiple of 16 bytes
    assert torch.equal(fa.paged_attention_fn(odd, kc, vc, table, n), fa.paged_attention_fn(odd.clone(), kc, vc, table, n))


def test_offsets_beyond_32_bits(device_ok):
    """Pages, heads and tokens that lie more than 2^32 elements into the cache."""
    page, Hkv, D = 16, 2, 64
    far = 2 ** 31 + 64
    room = torch.empty(2 * far + far // 2 + 2 ** 20, dtype=BF, device="cuda")
    kc = room.as_strided((3, page, Hkv, D), (far, Hkv * D, D, 1))
    vc = room[2 ** 18:].as_strided((3, page, Hkv, D), (far, Hkv * D, D, 1))
    g = torch.Generator(device="cuda").manual_seed(10)
    kc.copy_(torch.randn(kc.shape, device="cuda", generator=g))
    vc.copy_(torch.randn(vc.shape, device="cuda", generator=g))
    table = torch.tensor([[2, 0, 1], [1, 2, 0]], dtype=torch.int32, device="cuda")
    n = torch.tensor([48, 29], dtype=torch.int32, device="cuda")
    q = make_q(2, 4, D, BF, 10)
    check(fa.paged_attention_fn(q, kc, vc, table, n), q, kc, vc, table, n)
    rows = torch.randn(2, Hkv, D, device="cuda").to(BF)
    fa.paged_kv_write(rows, rows * 2, kc, vc, torch.tensor([47, 3], device="cuda"))
    assert torch.equal(kc[2, 15], rows[0]) and torch.equal(kc[0, 3], rows[1]) and torch.equal(vc[2, 15], rows[0] * 2)


@pytest.mark.parametrize("B,longest", [(1, 30000), (70, 900), (300, 40), (3000, 17)])
def test_splits_of_many_and_of_long_sequences(B, longest, device_ok):
    """The work of a call goes to the SMs in equal shares, whatever the lengths: shares that begin and end inside sequences,
    shares of many sequences, sequences of many shares, and the same bits when it is asked again."""
    lens = [longest - int((longest + 1) * (i * 0.618 % 1)) for i in range(B)]
    kc, vc, table, n = make_cache(lens, 16, 2, 64, BF, 11)
    q = make_q(B, 6, 64, BF, 11)
    got = fa.paged_attention_fn(q, kc, vc, table, n)
    check(got, q, kc, vc, table, n)
    for _ in range(3):
        assert torch.equal(fa.paged_attention_fn(q, kc, vc, table, n), got)


@pytest.mark.parametrize("most_ctas", ["1", "3", "20"])
@pytest.mark.parametrize("lens,page,Hkv,group,D", [([900, 0, 33, 2000], 16, 2, 4, 128), ([70] * 40, 8, 3, 2, 64),
                                                   ([500, 1200, 1], 20, 1, 10, 256), ([5, 700] * 30, 16, 8, 1, 32)])
def test_stretches_of_any_length(lens, page, Hkv, group, D, most_ctas, monkeypatch, device_ok):
    """With one, three and twenty CTAs: long stretches over many sequences, more sequences than stretches and fewer."""
    kc, vc, table, n = make_cache(lens, page, Hkv, D, BF, 15)
    q = make_q(len(lens), Hkv * group, D, BF, 15)
    monkeypatch.setenv("FA_MAX_CTAS", most_ctas)
    check(fa.paged_attention_fn(q, kc, vc, table, n), q, kc, vc, table, n)


@pytest.mark.parametrize("Hkv,group,D,longest", [(1, 3, 256, 20000), (8, 2, 128, 9000), (1, 20, 128, 6000), (5, 1, 16, 15000),
                                                 (1, 32, 64, 8000)])
def test_one_long_sequence(Hkv, group, D, longest, device_ok):
    """Hundreds of unfinished sums a head, of every width, for the joining kernel."""
    kc, vc, table, n = make_cache([longest], 16, Hkv, D, HF, 16)
    q = make_q(1, Hkv * group, D, HF, 16)
    check(fa.paged_attention_fn(q, kc, vc, table, n), q, kc, vc, table, n)


def test_caches_that_are_expanded_views(device_ok):
    """One page for all, one head for all: no tile map has them."""
    g = torch.Generator().manual_seed(17)
    page = torch.randn(1, 16, 2, 64, generator=g).to(BF).cuda()
    kc, vc = page.expand(5, 16, 2, 64), (page[:, :, :1] * 2).expand(5, 16, 2, 64)
    table, n = torch.tensor([[4, 0, 2]], dtype=torch.int32, device="cuda"), torch.tensor([41], dtype=torch.int32, device="cuda")
    q = make_q(1, 4, 64, BF, 17)
    check(fa.paged_attention_fn(q, kc, vc, table, n), q, kc, vc, table, n)


def test_inference_mode_and_no_grad(device_ok):
    with torch.inference_mode():
        kc, vc, table, n = make_cache([30, 5], 16, 1, 64, BF, 18)
        q = make_q(2, 2, 64, BF, 18)
        out = fa.paged_attention_fn(q, kc, vc, table, n)
        fa.paged_kv_write(kc[0, :2], vc[0, :2], kc, vc, torch.tensor([17, -1], device="cuda"))
    with torch.no_grad():
        kc, vc, table, n = make_cache([30, 5], 16, 1, 64, BF, 18)
        assert torch.equal(fa.paged_attention_fn(make_q(2, 2, 64, BF, 18).requires_grad_(), kc, vc, table, n), out)
    with pytest.raises(NotImplementedError):
        fa.paged_attention_fn(make_q(2, 2, 64, BF, 18).requires_grad_(), kc, vc, table, n)


def test_operators_are_captured_as_graph_nodes(device_ok):
    kc, vc, table, n = make_cache([30, 65], 16, 2, 64, BF, 19, stale=0.0)
    q, rows = make_q(2, 4, 64, BF, 19), make_q(2, 2, 64, BF, 20)
    slots = torch.tensor([table[0, 0].item() * 16 + 3, -1], device="cuda")
    k2, v2 = kc.clone(), vc.clone()
    fa.paged_kv_write(rows, rows, kc, vc, slots)
    want = fa.paged_attention_fn(q, kc, vc, table, n)
    seen = []

    def backend(gm, example_inputs):
        seen.append([node.target for node in gm.graph.nodes if node.op == "call_function"])
        return gm.forward

    def step(q, rows, k, v):
        fa.paged_kv_write_op(rows, rows, k, v, slots)
        return fa.paged_attention_op(q, k, v, table, n)

    with torch.no_grad():
        out = torch.compile(step, backend=backend, fullgraph=True)(q, rows, k2, v2)
    assert torch.equal(out, want) and torch.equal(k2, kc) and torch.equal(v2, vc)
    assert any(torch.ops.triton_flashattn_b200.paged_attn.default in g for g in seen)


def test_one_token_and_pages_shared_by_sequences(device_ok):
    kc, vc, table, n = make_cache([40], 16, 1, 128, BF, 12)
    table, n = table.expand(5, -1), torch.tensor([40, 1, 17, 0, 33], dtype=torch.int32, device="cuda")
    q = make_q(5, 2, 128, BF, 12)
    got = fa.paged_attention_fn(q, kc, vc, table, n)
    check(got, q, kc, vc, table, n)
    assert torch.equal(got[1], vc[table[1, 0], 0].expand(2, -1))  # one key: its value


def test_other_streams_and_graphs_that_overlap(device_ok):
    """Calls on a side stream; two captured graphs, replayed side by side many times over lengths that change, give what eager
    calls give."""
    sets = []
    for seed in (13, 14):
        kc, vc, table, n = make_cache([900, 411, 65], 16, 2, 128, BF, seed, stale=0.0)
        sets.append((make_q(3, 8, 128, BF, seed), kc, vc, table, n))
    want = {}
    for i, (q, kc, vc, table, n) in enumerate(sets):
        for cut in (1, 2, 5):
            want[i, cut] = fa.paged_attention_fn(q, kc, vc, table, n // cut)
    torch.cuda.synchronize()
    streams, graphs, outs, lens = [], [], [], []
    for q, kc, vc, table, n in sets:
        s = torch.cuda.Stream()
        live = n.clone()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            assert torch.equal(fa.paged_attention_fn(q, kc, vc, table, live), want[len(outs), 1])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(fa.paged_attention_fn(q, kc, vc, table, live))
        streams.append(s)
        graphs.append(g)
        lens.append(live)
    for cut in (1, 2, 5, 2, 1):
        torch.cuda.synchronize()
        for live, (_, _, _, _, n) in zip(lens, sets):
            live.copy_(n // cut)
        torch.cuda.synchronize()
        for _ in range(20):
            for s, g in zip(streams, graphs):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], want[i, cut])


def test_many_calls_in_flight(device_ok):
    """Calls of different sizes one after the other without a wait: what each gives alone."""
    sets = []
    for i, (lens, Hkv, group, D) in enumerate((([700, 20], 2, 4, 128), ([3] * 50, 1, 2, 64), ([5000], 1, 8, 128), ([90, 0, 80], 4, 1, 256))):
        kc, vc, table, n = make_cache(lens, 16, Hkv, D, BF, 20 + i)
        sets.append((make_q(len(lens), Hkv * group, D, BF, i), kc, vc, table, n))
    alone = []
    for s in sets:
        alone.append(fa.paged_attention_fn(*s))
        torch.cuda.synchronize()
    got = [fa.paged_attention_fn(*s) for _ in range(10) for s in sets]
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert torch.equal(g, alone[i % len(sets)])


def test_no_store_outside_the_result(device_ok):
    """Through the C entry, with the result in strided rows between sentinels and a workspace of just its size."""
    lib = _cabi.load()
    for lens, Hkv, group, D in (([700, 20, 0], 2, 5, 128), ([90] * 40, 1, 1, 16), ([2500], 1, 12, 256), ([77, 200], 2, 2, 32)):
        kc, vc, table, n = make_cache(lens, 16, Hkv, D, BF, 30)
        B, H = len(lens), Hkv * group
        q = make_q(B, H, D, BF, 30)
        room = torch.full((B + 2, H + 1, D + 8), 77.0, dtype=BF, device="cuda")
        out = room[1:-1, :H, :D]
        p = _cabi.FaPagedParams()
        p.struct_size, p.device = ctypes.sizeof(p), 0
        p.B, p.H, p.Hkv, p.D, p.page_size, p.width, p.num_pages = B, H, Hkv, D, 16, table.shape[1], kc.shape[0]
        p.dtype, p.bias_kind, p.sm_scale = 1, 0, D ** -0.5
        p.q, p.k_cache, p.v_cache, p.o = q.data_ptr(), kc.data_ptr(), vc.data_ptr(), out.data_ptr()
        p.block_table, p.seq_lens, p.table_stride = table.data_ptr(), n.data_ptr(), table.stride(0)
        p.q_stride, p.o_stride = _cabi._I64x2(*q.stride()[:2]), _cabi._I64x2(*out.stride()[:2])
        p.k_stride = p.v_stride = _cabi._I64x3(*kc.stride()[:3])
        size = lib.fa_paged_workspace_bytes(ctypes.byref(p))
        guard = 4096
        ws = torch.full((size + 2 * guard,), 91, dtype=torch.uint8, device="cuda")
        stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
        if size:
            assert lib.fa_paged_fwd(ctypes.byref(p), ws.data_ptr() + guard, size - 1, stream) == 2  # too little
        assert lib.fa_paged_fwd(ctypes.byref(p), ws.data_ptr() + guard, size, stream) == 0
        torch.cuda.synchronize()
        assert (ws[:guard] == 91).all() and (ws[guard + size:] == 91).all()
        assert torch.equal(out, fa.paged_attention_fn(q, kc, vc, table, n))
        room[1:-1, :H, :D] = 77.0
        assert (room == 77.0).all()


def test_refusals_on_the_device(device_ok):
    kc, vc, table, n = make_cache([30], 16, 1, 64, BF, 31)
    q = make_q(1, 2, 64, BF, 31)
    for bias, error in ((torch.zeros(1, 2, 31, device="cuda"), ValueError), (torch.zeros(1, 2, 32), ValueError),
                        (torch.zeros(1, 2, 32, dtype=torch.int32, device="cuda"), TypeError)):
        with pytest.raises(error):
            fa.paged_attention_fn(q, kc, vc, table, n, bias)
    with pytest.raises(ValueError, match="block_table"):
        fa.paged_attention_fn(q, kc, vc, table.cpu(), n)
    with pytest.raises(ValueError, match="seq_lens"):
        fa.paged_attention_fn(q, kc, vc, table, n.cpu())
    with pytest.raises((TypeError, ValueError)):
        fa.paged_attention_fn(q, kc, vc, table, n, None, "x")
    assert fa.paged_attention_fn(q[:0], kc, vc, table[:0], n[:0]).shape == (0, 2, 64)
    with pytest.raises(ValueError, match="new_lens"):
        fa.paged_kv_extend(table, n, n.cpu(), torch.zeros(4, dtype=torch.int32, device="cuda"), n, 16, 4)
    with pytest.raises(ValueError, match="rows of their own"):
        fa.paged_kv_extend(table.expand(3, -1), n.expand(3), n.expand(3), torch.zeros(4, dtype=torch.int32, device="cuda"), n, 16, 4)
    with pytest.raises(ValueError, match="dense"):
        two = torch.stack([n, n], 1).expand(1, 2)
        fa.paged_kv_extend(table.expand(2, -1).clone(), torch.zeros(4, dtype=torch.int32, device="cuda")[::2], two[0],
                           torch.zeros(4, dtype=torch.int32, device="cuda"), n, 16, 4, inplace=True)
    with pytest.raises(ValueError, match="negative"):
        fa.paged_kv_extend(table, n, n, torch.zeros(4, dtype=torch.int32, device="cuda"), n, 16, -1)


# ---------------------------------------------------------------------------------- rows
@pytest.mark.parametrize("T,Hkv,D,page,dtype", [(1, 1, 16, 16, BF), (7, 3, 32, 1, HF), (64, 8, 128, 16, BF), (300, 2, 64, 7, HF),
                                                (1000, 1, 256, 48, BF), (4097, 5, 128, 128, BF)])
@pytest.mark.parametrize("layout", ["dense", "sliced", "heads_first"])
def test_rows_go_where_their_slots_say(T, Hkv, D, page, dtype, layout, device_ok):
    g = torch.Generator().manual_seed(40)
    pages = -(-T // page) + 2
    k, v = (torch.randn(T, Hkv, D, generator=g).to(dtype).cuda() for _ in range(2))
    if layout == "sliced":  # slices of one projection, at any address
        qkv = torch.randn(T * (4 * Hkv) * D + 1, generator=g).to(dtype).cuda()
        qkv = (qkv[1:] if T % 2 else qkv[:-1]).view(T, 4 * Hkv, D)
        k, v = qkv[:, 2 * Hkv:3 * Hkv], qkv[:, 3 * Hkv:]
    kc, vc = (torch.randn(pages, page, Hkv, D, generator=g).to(dtype).cuda() for _ in range(2))
    if layout == "heads_first":
        kc, vc = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (kc, vc))
    slots = torch.randperm(pages * page, generator=g)[:T]
    slots[::5] = torch.tensor([-1, pages * page, -2 ** 63, 2 ** 62, -page])[torch.arange(len(slots[::5])) % 5]
    want_k, want_v = kc.clone(), vc.clone()
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            want_k[s // page, s % page], want_v[s // page, s % page] = k[t], v[t]
    before = kc._version
    fa.paged_kv_write(k, v, kc, vc, slots.cuda())
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)
    assert kc._version > before
    fa.paged_kv_write(k[:0], v[:0], kc, vc, slots[:0].cuda())
    assert torch.equal(kc, want_k)


def test_row_writes_stay_inside_the_cache(device_ok):
    room = torch.full((6, 17, 3, 40), 5.0, dtype=BF, device="cuda")
    kc, vc = room[1:3, :16, :2, :32], room[4:, :16, :2, :32]  # room for nothing else
    with torch.no_grad():
        k = torch.randn(40, 2, 32, device="cuda").to(BF).requires_grad_()
        fa.paged_kv_write(k, k, kc, vc, torch.arange(-4, 36, device="cuda"))
    assert torch.equal(kc.reshape(32, 2, 32), k[4:36]) and torch.equal(vc.reshape(32, 2, 32), k[4:36])
    kc.fill_(5.0), vc.fill_(5.0)
    assert (room == 5.0).all()


# ---------------------------------------------------------------------------------- tables
def extend_ref(table, lens, new, stack, count, page, T):
    table, lens, new, stack = [r[:] for r in table], lens[:], new[:], stack[:]
    width, slots, off, short = len(table[0]), [-1] * T, 0, False
    wanted, taken = 0, 0
    for b in range(len(lens)):
        n, old = max(new[b], 0), max(lens[b], 0)
        at, off = off, off + n
        if old + n > width * page or off > T:
            continue
        have = -(-old // page)
        need = -(-(old + n) // page) - have
        short = short or (need > 0 and wanted + need > count)
        wanted += need
        if need > 0 and short:
            continue
        for j in range(need):
            table[b][have + j] = stack[count - 1 - taken]
            taken += 1
        for i in range(n):
            page_id = table[b][(old + i) // page]
            slots[at + i] = page_id * page + (old + i) % page if page_id >= 0 else -1
        lens[b] = old + n
    return table, slots, lens, count - taken


def release_ref(table, lens, finished, stack, count, page):
    lens, stack = lens[:], stack[:]
    for b in range(len(lens)):
        if finished[b]:
            for j in range(min(-(-max(lens[b], 0) // page), len(table[b]))):
                if count < len(stack):
                    stack[count] = table[b][j]
                    count += 1
            lens[b] = 0
    return lens, stack, count


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("B,page,width,longest,most_new,pages,T,seed", [
    (1, 16, 4, 20, 1, 8, 1, 0), (3, 16, 8, 40, 30, 40, 90, 1), (3, 16, 8, 40, 30, 7, 90, 2), (5, 1, 30, 9, 9, 100, 45, 3),
    (40, 8, 12, 60, 50, 120, 900, 4), (513, 16, 9, 100, 1, 6000, 513, 5), (1500, 4, 20, 40, 30, 9000, 30000, 6),
    (1500, 4, 20, 40, 30, 15000, 9000, 7), (600, 16, 6, 90, 12, 2800, 9000, 8), (2, 128, 40, 3, 5000, 90, 10000, 9),
    (30, 16, 5, 100, 0, 200, 3, 10)])
@pytest.mark.parametrize("inplace", [False, True])
def test_tables_and_slots_against_a_plain_loop(B, page, width, longest, most_new, pages, T, seed, inplace, device_ok):
    """One request and thousands, requests that outgrow their row, a stack that runs out, too few rows for all tokens, lengths
    below zero; then the pages of some of them go back."""
    g = torch.Generator().manual_seed(seed)
    r = lambda lo, hi, n: torch.randint(lo, hi + 1, (n,), generator=g).tolist()  # noqa: E731
    lens, new = r(0, min(longest, width * page), B), r(-1 if B > 10 else 0, most_new, B)
    if B > 20:
        lens[3], lens[7] = -4, width * page
    table = [r(0, 10 ** 6, width) for _ in range(B)]
    if B > 20:
        table[5][0] = -3  # no page: its tokens there have no slot
    stack, count = r(0, 10 ** 6, pages), pages * 3 // 4 if pages > 50 else pages
    want = extend_ref(table, lens, new, stack, count, page, T)
    room = torch.full((B, width + 3), -9, dtype=torch.int32, device="cuda")
    t, ln, st, c = room[:, :width], ints(lens), ints(stack), ints([count])
    t.copy_(ints(table))
    slots, after, left = fa.paged_kv_extend(t, ln, ints(new), st, c, page, T, inplace)
    assert slots.dtype == torch.int64 and slots.tolist() == want[1]
    assert t.tolist() == want[0] and (room[:, width:] == -9).all()
    assert after.tolist() == want[2] and left.tolist() == [want[3]] and st.tolist() == stack
    if inplace:
        assert after.data_ptr() == ln.data_ptr() and left.data_ptr() == c.data_ptr()
    else:
        assert ln.tolist() == lens and c.tolist() == [count]
        again = fa.paged_kv_extend(t, ln, ints(new), st, c, page, T)
        assert again[0].tolist() == want[1] and t.tolist() == want[0]
    finished = [x == 0 for x in r(0, 2, B)]
    back = release_ref(want[0], want[2], finished, stack, want[3], page)
    gone = torch.tensor(finished, device="cuda")
    ln2, c2 = fa.paged_kv_release(t, after, gone, st, left, page, inplace)
    assert ln2.tolist() == back[0] and st.tolist() == back[1] and c2.tolist() == [back[2]]
    assert t.tolist() == want[0]
    if inplace:
        assert ln2.data_ptr() == ln.data_ptr() and c2.data_ptr() == c.data_ptr()


def test_tables_at_their_ends(device_ok):
    empty = torch.empty(0, dtype=torch.int32, device="cuda")
    t0 = torch.empty(0, 4, dtype=torch.int32, device="cuda")
    slots, lens, count = fa.paged_kv_extend(t0, empty, empty, empty, ints([0]), 16, 5)
    assert slots.tolist() == [-1] * 5 and lens.shape == (0,) and count.tolist() == [0]
    t1, st = ints([[4, 5]]), ints([9, 8, 7])
    assert fa.paged_kv_extend(t1, ints([16]), ints([0]), st, ints([3]), 16, 0)[0].shape == (0,)
    # a count beyond the stack's ends is cut to them
    slots, lens, count = fa.paged_kv_extend(t1, ints([16]), ints([1]), st, ints([100]), 16, 1)
    assert slots.tolist() == [7 * 16] and t1.tolist() == [[4, 7]] and count.tolist() == [2]
    slots, lens, count = fa.paged_kv_extend(t1, ints([16]), ints([1]), st, ints([-3]), 16, 1)
    assert slots.tolist() == [-1] and lens.tolist() == [16] and count.tolist() == [0]
    big = torch.iinfo(torch.int32).max
    slots, lens, count = fa.paged_kv_extend(t1, ints([big]), ints([big]), st, ints([3]), 16, 4)
    assert slots.tolist() == [-1] * 4 and lens.tolist() == [big] and count.tolist() == [3]
    yes = torch.tensor([True], device="cuda")
    assert fa.paged_kv_release(t1, ints([big]), yes, st, ints([1]), 16)[1].tolist() == [3] and st.tolist() == [9, 4, 7]
    lens, count = fa.paged_kv_release(t1, ints([32]), yes, st, ints([2]), 16)  # one place left
    assert count.tolist() == [3] and st.tolist() == [9, 4, 4]


# ---------------------------------------------------------------------------------- together
@pytest.mark.parametrize("dtype,Hkv,group,D,page", [(BF, 2, 4, 64, 16), (HF, 1, 1, 128, 24)])
@pytest.mark.parametrize("captured", [False, True])
def test_a_server_loop_against_dense_attention(dtype, Hkv, group, D, page, captured, device_ok):
    """Prompts through the dense causal forward, their keys into the cache, then tokens one by one (eager, or one captured step
    replayed), a request that ends and another that takes its place and its pages: each step's results against 64 bits over
    the keys that were fed in, and the prompts' last tokens against the dense forward."""
    H, layers, seqs, max_len = Hkv * group, 2, 4, 200
    g = torch.Generator().manual_seed(50)
    cache = fa.PagedKVCache(layers, 22, page, Hkv, D, seqs, max_len, dtype)
    cache.k.fill_(float("nan")), cache.v.fill_(float("nan"))
    fed = [[([], []) for _ in range(seqs)] for _ in range(layers)]

    def feed(new):
        T = sum(new)
        slots = cache.extend(ints(new), T)
        kv = []
        for layer in range(layers):
            k, v = (torch.randn(T, Hkv, D, generator=g).to(dtype).cuda() for _ in range(2))
            cache.write(layer, k, v, slots)
            at = 0
            for b, n in enumerate(new):
                fed[layer][b][0].extend(k[at:at + n]), fed[layer][b][1].extend(v[at:at + n])
                at += n
            kv.append((k, v))
        return kv

    def expect(layer, q):
        n = [len(fed[layer][b][0]) for b in range(seqs)]
        assert cache.seq_lens.tolist() == n
        kc, vc = (torch.zeros(seqs, max(n), Hkv, D, dtype=dtype, device="cuda") for _ in range(2))
        for b in range(seqs):
            if n[b]:
                kc[b, :n[b]], vc[b, :n[b]] = torch.stack(fed[layer][b][0]), torch.stack(fed[layer][b][1])
        return attend_ref(q, kc, vc, torch.arange(seqs)[:, None], ints(n))  # a page a sequence

    prompts = [37, 1, 100, 0]
    kv = feed(prompts)
    q_all = torch.randn(sum(prompts), H, D, generator=g).to(dtype).cuda()
    last = torch.zeros(seqs, H, D, dtype=dtype, device="cuda")
    at = 0
    for b, n in enumerate(prompts):
        if n:
            last[b] = q_all[at + n - 1]
        at += n
    for layer in range(layers):
        out = cache.attend(layer, last)
        ref, tol = expect(layer, last)
        assert ((out.double().cpu() - ref).abs() <= tol).all()
        assert not out[3].any()
        at = 0
        for b, n in enumerate(prompts):
            if n:
                q1, k1, v1 = (t[at:at + n].unsqueeze(0) for t in (q_all, *kv[layer]))
                dense = fa.flash_attention_fn(q1, k1.repeat_interleave(group, 2), v1.repeat_interleave(group, 2), None, True)[0, -1]
                # both within their tolerances of the same value; the dense forward rounds its weights to 16 bits once: u sum w |v|
                u = torch.finfo(dtype).eps / 2
                gap = (out[b].double() - dense.double()).abs().cpu()
                assert (gap <= 2 * tol[b] + 2 * u * v1.double().abs().max().cpu()).all()
            at += n

    step = {name: torch.zeros(shape, dtype=dtype, device="cuda") for name, shape in
            (("q", (seqs, H, D)), ("k", (layers, seqs, Hkv, D)), ("v", (layers, seqs, Hkv, D)))}
    new = ints([0] * seqs)

    def run():
        slots = cache.extend(new, seqs)
        outs = []
        for layer in range(layers):
            cache.write(layer, step["k"][layer], step["v"][layer], slots)
            outs.append(cache.attend(layer, step["q"]))
        return outs

    graph = None
    if captured:
        run()  # (nothing new: nothing changes)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = run()
    for i in range(40):
        if i == 17:  # one ends, and another takes its place
            done = torch.tensor([False, False, True, False], device="cuda")
            cache.release(done)
            for layer in range(layers):
                fed[layer][2] = ([], [])
            feed([0, 0, 60, 33])
        active = [b for b in range(seqs) if len(fed[0][b][0])]
        for t in step.values():
            t.copy_(torch.randn(t.shape, generator=g))
        new.copy_(ints([1 if b in active else 0 for b in range(seqs)]))
        for layer in range(layers):
            for row, b in enumerate(active):
                fed[layer][b][0].append(step["k"][layer][row].clone()), fed[layer][b][1].append(step["v"][layer][row].clone())
        if captured:
            graph.replay()
        else:
            outs = run()
        for layer in range(layers):
            ref, tol = expect(layer, step["q"])
            assert ((outs[layer].double().cpu() - ref).abs() <= tol).all(), (i, layer)
    held = sum(-(-n // page) for n in cache.seq_lens.tolist())
    assert cache.free_count.item() == 22 - held
    pages = [p for b in range(seqs) for p in cache.block_table[b, :-(-cache.seq_lens[b].item() // page)].tolist()]
    assert sorted(pages + cache.free_pages[:cache.free_count.item()].tolist()) == list(range(22))
