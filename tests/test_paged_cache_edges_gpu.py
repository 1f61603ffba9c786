"""GPU tests of the paged cache at its edges: what a bias of -inf leaves out, calls that want a derivative, scores at the end
of what fp32 tells apart."""
import pytest
import torch

import triton_flashattn_b200 as fa
from tests.test_paged_cache_gpu import BF, HF, INF, check, make_cache, make_q

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


# ---------------------------------------------------------------------------------- weights
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
