"""GPU tests of the paged cache at its edges: what a bias of -inf leaves out, calls that want a derivative, memory that a
bias takes, rows of the cache itself, weights far below the largest one, scores at the end of what fp32 tells apart,
sequences that are not split."""
import pytest
import torch

import triton_flashattn_b200 as fa
from tests.test_paged_cache_gpu import BF, HF, INF, check, make_cache, make_q
from triton_flashattn_b200 import _cabi

pytestmark = pytest.mark.gpu

NAN = float("nan")


@pytest.mark.parametrize("lens,page,Hkv,group,D,dtype", [([100, 1, 777, 0], 16, 2, 4, 128, BF), ([130, 55], 24, 1, 10, 64, HF),
                                                         ([300, 20], 32, 2, 2, 256, BF), ([90, 400], 5, 2, 3, 32, HF),
                                                         ([40, 210], 8, 1, 20, 128, BF), ([60, 3], 16, 2, 2, 64, HF)])
@pytest.mark.parametrize("kind", ["same", "f32", "table", "f64"])
def test_a_bias_of_minus_infinity_leaves_out_any_key(lens, page, Hkv, group, D, dtype, kind, device_ok):
    """Keys and values that are infinite or NaN behind a bias of -inf: the same bits as with finite ones there.  One head has
    nothing but -inf, one a single key; and where one head alone looks at a NaN key, the others do not see it."""
    kc, vc, table, n = make_cache(lens, page, Hkv, D, dtype, 60)
    B, H, N = len(lens), Hkv * group, table.shape[1] * page
    q = make_q(B, H, D, dtype, 60)
    g = torch.Generator().manual_seed(61)
    x = torch.randn(B, H, N, generator=g)
    hidden = torch.rand(N, generator=g) < 0.3
    hidden[0], hidden[1:3] = False, True
    if kind == "table":
        x = x[:1]
    x[:, :, hidden] = -INF
    x[:, 0, 1:] = -INF
    x[:, 1] = -INF
    bias = x.cuda().to({"same": dtype, "f32": torch.float32, "table": torch.float32, "f64": torch.float64}[kind]).expand(B, H, N)
    clean = fa.paged_attention_fn(q, kc, vc, table, n, bias)
    check(clean, q, kc, vc, table, n, bias.float() if kind == "f64" else bias)
    assert not clean[:, 1].any()
    for b, length in enumerate(lens):
        for i, at in enumerate(hidden[:length].nonzero()[:, 0].tolist()):
            row = table[b, at // page], at % page
            kc[row], vc[row] = (NAN, INF, -INF)[i % 3], (1.0, NAN, INF, -INF)[i % 4]
            if i % 5 == 0:  # scores of +inf, -inf and NaN beside one another
                kc[row] = torch.where(torch.arange(D, device="cuda") < D // 2, INF, 0.0).to(dtype)
    assert torch.equal(fa.paged_attention_fn(q, kc, vc, table, n, bias), clean)
    # the last head alone sees position 0, where a NaN key comes to lie
    alone = bias.clone()
    alone[:, :, 0], alone[:, -1, 0] = -INF, 0.0
    others = fa.paged_attention_fn(q, kc, vc, table, n, alone)
    for b, length in enumerate(lens):
        if length:
            kc[table[b, 0], 0] = NAN
    seen = fa.paged_attention_fn(q, kc, vc, table, n, alone)
    assert torch.equal(seen[:, :-1], others[:, :-1])
    for b, length in enumerate(lens):
        assert seen[b, -1].isnan().all() if length else not seen[b].any()


# ---------------------------------------------------------------------------------- operators without a derivative
def test_operators_refuse_what_would_lose_a_derivative(device_ok):
    """Grad, functorch's grad and a tangent: refused before anything is written."""
    kc, vc, table, n = make_cache([30, 5], 16, 1, 64, BF, 62, stale=0.0)
    q, rows = make_q(2, 2, 64, BF, 62), make_q(2, 1, 64, BF, 63)
    slots = torch.tensor([17, 3], device="cuda")
    before = kc.clone(), vc.clone()
    for wants in ((rows.clone().requires_grad_(), rows), (rows, rows.clone().requires_grad_())):
        with pytest.raises(NotImplementedError, match="no backward"):
            fa.paged_kv_write_op(*wants, kc, vc, slots)
        with pytest.raises(NotImplementedError, match="no backward"):
            torch.ops.triton_flashattn_b200.paged_kv_write(*wants, kc, vc, slots)
    for i in range(3):
        a = [q, kc, vc]
        a[i] = a[i].clone().requires_grad_()
        with pytest.raises(NotImplementedError, match="no backward"):
            fa.paged_attention_op(*a, table, n)
    with pytest.raises(NotImplementedError, match="no backward"):
        fa.paged_attention_op(q, kc, vc, table, n, torch.zeros(2, 2, table.shape[1] * 16, device="cuda", requires_grad=True))

    def through(k):
        fa.paged_kv_write_op(k, rows, kc, vc, slots)
        return kc.float().sum()

    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.grad(through)(rows)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.grad(lambda q: fa.paged_attention_op(q, kc, vc, table, n).float().sum())(q)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(rows, rows)
        with pytest.raises((NotImplementedError, RuntimeError)):
            fa.paged_kv_write_op(dual, rows, kc, vc, slots)
        with pytest.raises((NotImplementedError, RuntimeError)):
            fa.paged_attention_op(torch.autograd.forward_ad.make_dual(q, q), kc, vc, table, n)
    assert torch.equal(kc, before[0]) and torch.equal(vc, before[1])
    with torch.no_grad():
        leaf = rows.clone().requires_grad_()
        version = kc._version
        fa.paged_kv_write_op(leaf, leaf, kc, vc, slots)
        assert kc._version > version and torch.equal(kc[1, 1], rows[0]) and torch.equal(vc[0, 3], rows[1])
        want = fa.paged_attention_fn(q, kc, vc, table, n)
        assert torch.equal(fa.paged_attention_op(q.clone().requires_grad_(), kc, vc, table, n), want)
    assert torch.equal(fa.paged_attention_op(q, kc, vc, table, n), want)


# ---------------------------------------------------------------------------------- biases that are converted
@pytest.mark.parametrize("what", ["fp64 table", "fp16 a head", "fp64 a sequence", "fp32 every other", "mask every other", "one number"])
def test_expanded_biases_are_not_written_out(what, device_ok):
    """A bias that has to be converted, or laid out anew, and is expanded over the batch or the heads: a copy of what there is of
    it, not of the (B, H, N) that it stands for."""
    B, H, page, width = 12, 32, 16, 64
    N = page * width
    kc, vc, table, n = make_cache([700 - 50 * i for i in range(B)], page, 8, 64, BF, 64, width=width)
    q = make_q(B, H, 64, BF, 64)
    x = torch.randn(B, H, 2 * N, generator=torch.Generator().manual_seed(65)).to(HF).cuda()
    bias = {"fp64 table": lambda: x[:1, :1, :N].double(), "fp16 a head": lambda: x[:1, :, :N].clone(),
            "fp64 a sequence": lambda: x[:, :1, :N].double(), "fp32 every other": lambda: x[:1, :1].float()[:, :, ::2],
            "mask every other": lambda: (x[:, :1] > 0)[:, :, ::2], "one number": lambda: x[:1, :1, :1].to(BF)}[what]().expand(B, H, N)
    full = bias.contiguous()  # (as it is, or in fp32 for another dtype)
    want = fa.paged_attention_fn(q, kc, vc, table, n, full if full.dtype in (torch.bool, BF) else full.float())
    fa.paged_attention_fn(q, kc, vc, table, n)
    torch.cuda.synchronize()

    def peak(bias):
        torch.cuda.reset_peak_memory_stats()
        start = torch.cuda.memory_allocated()
        out = fa.paged_attention_fn(q, kc, vc, table, n, bias)
        return out, torch.cuda.max_memory_allocated() - start

    plain = peak(None)[1]  # result and workspace
    got, used = peak(bias)
    assert torch.equal(got, want)
    # at most one fp32 number an element of the largest of them, (1, H, N), in blocks of 512 bytes
    assert used - plain <= 4 * H * N + 512


# ---------------------------------------------------------------------------------- rows of the cache itself
@pytest.mark.parametrize("Hkv,D,page", [(8, 128, 16), (1, 16, 7), (3, 256, 64)])
@pytest.mark.parametrize("by", [1, -1, 0, 1000])
def test_rows_that_lie_in_the_cache_are_moved_as_they_were(Hkv, D, page, by, device_ok):
    """Rows read from slots that the same call writes: each slot gets what its source held before the call."""
    pages = -(-5000 // page)
    g = torch.Generator().manual_seed(66)
    kc, vc = (torch.randn(pages, page, Hkv, D, generator=g).to(BF).cuda() for _ in range(2))
    total = pages * page
    src = torch.arange(total)
    slots = (src + by) % total if by >= 0 else src + by  # (one of them then has no slot)
    want_k, want_v = kc.clone(), vc.clone()
    has = slots >= 0
    # k out of the values and v out of the keys
    want_k.view(total, Hkv, D)[slots[has].cuda()] = vc.view(total, Hkv, D)[src[has].cuda()]
    want_v.view(total, Hkv, D)[slots[has].cuda()] = kc.view(total, Hkv, D)[src[has].cuda()]
    fa.paged_kv_write(vc.view(total, Hkv, D), kc.view(total, Hkv, D), kc, vc, slots.cuda())
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)


def test_a_page_is_copied_to_another_one(device_ok):
    kc, vc, table, n = make_cache([48], 16, 2, 64, HF, 67, stale=0.0)
    to = next(i for i in range(kc.shape[0]) if i not in table[0].tolist())
    fa.paged_kv_write(kc[table[0, 1]], vc[table[0, 1]], kc, vc, torch.arange(to * 16, to * 16 + 16, device="cuda"))
    assert torch.equal(kc[to], kc[table[0, 1]]) and torch.equal(vc[to], vc[table[0, 1]])
    q = make_q(1, 4, 64, HF, 67)
    want = fa.paged_attention_fn(q, kc, vc, table, n)
    fork = table.clone()
    fork[0, 1] = to
    assert torch.equal(fa.paged_attention_fn(q, kc, vc, fork, n), want)


# ---------------------------------------------------------------------------------- weights
@pytest.mark.parametrize("n,D,group,most_ctas", [(65536, 64, 4, "1"), (30011, 128, 1, "1"), (9000, 256, 12, "1"), (200000, 32, 2, "2")])
@pytest.mark.parametrize("below", [12.3, 17.9, 20.6])
@pytest.mark.parametrize("kind", ["none", "mask", "same", "f32"])
def test_one_strong_key_and_many_weak_ones(n, D, group, most_ctas, below, kind, monkeypatch, device_ok):
    """fp16: one key at the front, whose value is 0, and thousands whose weights are e^-below of its: what these add up to is all
    there is in the result.

    The tolerance, relative to sum w |v| (w the normalised weights): a score is exact up to its product with the scale and, with
    no bias, log2 e, and so is the difference of two: 2^-22 (|s| + |max|); the exponential adds 2^-21, numerator and
    sum have both: twice.  Sums of n keys in fp32, in both: 2 (n + 64) 2^-24.  Absolute: a weight enters the product in two fp16
    terms, the second rounded to half of fp16's smallest step, 2^-25, in units of 2^-7 of a weight of 1, and weights are at least the
    true ones beside the largest: 2^-32 a key over the sum of the weights; the result's own rounding 2^-11 relative, and not
    below 2^-25."""
    monkeypatch.setenv("FA_MAX_CTAS", most_ctas)
    page = 16
    pages = -(-n // page)
    g = torch.Generator().manual_seed(70)
    kc = torch.zeros(pages, page, 1, D, dtype=HF, device="cuda")
    vc = torch.zeros(pages, page, 1, D, dtype=HF, device="cuda")
    v = (1 + torch.rand(D, generator=g)).to(HF).cuda()
    vc[:] = v
    vc[0, 0] = 0.0
    q = torch.zeros(1, group, D, dtype=HF, device="cuda")
    q[:, :, 0] = 1.0
    table = torch.randperm(pages - 1, generator=g).int()[None] + 1
    table = torch.cat([torch.zeros(1, 1, dtype=torch.int32), table], 1).cuda()
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    bias, scale = None, 1.0
    if kind in ("none", "mask"):
        kc[0, 0, 0, 0] = below  # (rounded to fp16: taken from there below)
        gap = kc[0, 0, 0, 0].double().item()
        if kind == "mask":
            bias = torch.ones(1, 1, pages * page, dtype=torch.bool, device="cuda").expand(1, group, -1)
    else:
        row = torch.full((1, 1, pages * page), -below, dtype=HF if kind == "same" else torch.float32, device="cuda")
        gap = -row[0, 0, 0].double().item()
        row[:, :, 0] = 0.0
        bias = row.expand(1, group, -1)
    w = torch.exp(torch.tensor(-gap, dtype=torch.float64))
    total = 1 + (n - 1) * w
    share = (n - 1) * w / total  # sum w over the keys whose value is not 0
    want = share * v.double().cpu()
    rel = 2 * (2.0 ** -22 * 2 * gap + 2.0 ** -21) + 2 * (n + 64) * 2.0 ** -24
    tol = (2.0 ** -11 + rel) * want + n * 2.0 ** -32 / total * v.double().cpu().max() + 2.0 ** -25
    off = (fa.paged_attention_fn(q, kc, vc, table, lens, bias, scale)[0].double().cpu() - want).abs()
    assert (off <= tol).all(), f"{(off / want).max().item():.3e} of the result, {(off / tol).max().item():.2f} of the tolerance"


@pytest.mark.parametrize("first", [2.0 ** 27 + 16, -(2.0 ** 27 + 48)])
@pytest.mark.parametrize("D", [64, 256])
def test_scores_so_large_that_fp32_steps_by_16(first, D, monkeypatch, device_ok):
    """fp16 with an fp32 bias whose neighbours are 16 apart: the next score up has e^16 times the weight, beyond fp16, unless the
    running maximum moves."""
    monkeypatch.setenv("FA_MAX_CTAS", "1")
    kc, vc, table, n = make_cache([1000], 16, 1, D, HF, 71)
    q = torch.zeros(1, 3, D, dtype=HF, device="cuda")
    pos = torch.arange(table.shape[1] * 16, device="cuda")
    bias = (first + 16.0 * (pos // 32 % 2)).float().expand(1, 3, -1)
    check(fa.paged_attention_fn(q, kc, vc, table, n, bias), q, kc, vc, table, n, bias)


# ---------------------------------------------------------------------------------- sequences that are not split
@pytest.mark.parametrize("B,width,Hkv,group,D,launches", [
    (1, 1, 2, 16, 256, 1), (40, 1, 2, 16, 256, 1), (700, 1, 1, 12, 256, 1),  # one tile: nothing to split, whatever the warps share
    (1, 2, 1, 1, 64, 1), (300, 2, 3, 2, 32, 1), (5, 1, 1, 20, 128, 1), (33, 1, 5, 1, 128, 1),
    (200, 4, 8, 2, 128, 1), (1, 3, 8, 4, 128, 1), (147, 4, 12, 1, 64, 1),  # up to 64 keys, a unit for each warp
    (140, 4, 2, 16, 256, 1), (1, 4, 1, 8, 128, 1),  # or no more sequences than CTAs
    (200, 4, 2, 16, 256, 2), (200, 3, 1, 8, 128, 2), (200, 5, 8, 2, 128, 2)])
def test_sequences_that_are_not_split(B, width, Hkv, group, D, launches, device_ok):
    """One launch where no sequence can be split or none has to be, else two; pages that are not there among them."""
    lib = _cabi.load()
    g = torch.Generator().manual_seed(72)
    lens = torch.randint(0, width * 16 + 1, (B,), generator=g).tolist()
    lens[0] = width * 16
    for dtype in (BF, HF):
        kc, vc, table, n = make_cache(lens, 16, Hkv, D, dtype, 73, width=width)
        if B > 3:
            table[2, 0] = -1
        q = make_q(B, Hkv * group, D, dtype, 73)
        before = lib.fa_launch_count()
        out = fa.paged_attention_fn(q, kc, vc, table, n)
        if torch.cuda.get_device_properties(0).multi_processor_count == 148:
            assert lib.fa_launch_count() - before == launches
        check(out, q, kc, vc, table, n)
