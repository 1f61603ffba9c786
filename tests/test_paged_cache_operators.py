"""The paged cache's torch.library operators refuse inputs that want a gradient, as the functions do (CPU: shape-only tensors)."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import triton_flashattn_b200 as fa

BF = torch.bfloat16


def _args(which):
    cache = lambda: torch.empty(9, 16, 2, 64, dtype=BF, device="cuda")  # noqa: E731
    if which == "paged_attn":
        return dict(q=torch.empty(2, 8, 64, dtype=BF, device="cuda"), k_cache=cache(), v_cache=cache(),
                    block_table=torch.empty(2, 4, dtype=torch.int32, device="cuda"),
                    seq_lens=torch.empty(2, dtype=torch.int32, device="cuda"),
                    bias=torch.empty(2, 8, 64, device="cuda"), sm_scale=0.125)
    return dict(k=torch.empty(5, 2, 64, dtype=BF, device="cuda"), v=torch.empty(5, 2, 64, dtype=BF, device="cuda"), k_cache=cache(),
                v_cache=cache(), slot_mapping=torch.empty(5, dtype=torch.int64, device="cuda"))


@pytest.mark.parametrize("which,wrapper", [("paged_attn", fa.paged_attention_op), ("paged_kv_write", fa.paged_kv_write_op)])
def test_operators_refuse_inputs_that_want_a_gradient(which, wrapper):
    op = getattr(torch.ops.triton_flashattn_b200, which)
    with FakeTensorMode():
        floats = [n for n, t in _args(which).items() if isinstance(t, torch.Tensor) and t.is_floating_point()]
        assert len(floats) == 4
        for name in floats:
            a = _args(which)
            a[name].requires_grad_()
            for call in (lambda: wrapper(**a), lambda: op(**a), lambda: op(*a.values()), lambda: op.default(**a)):
                with pytest.raises(NotImplementedError, match="no backward"):
                    call()
            with torch.no_grad():
                out = wrapper(**a)
                assert out is None or (out.shape == a["q"].shape and not out.requires_grad)
        a = _args(which)
        out = wrapper(**a)  # nothing wants a gradient: no matter what grad mode is on
        assert out is None or not out.requires_grad
        with torch.inference_mode():
            wrapper(**a)


def test_a_traced_call_refuses_too():
    def step(k, v, kc, vc, slots):
        fa.paged_kv_write_op(k, v, kc, vc, slots)
        return kc

    with FakeTensorMode(allow_non_fake_inputs=True):
        a = _args("paged_kv_write")
        a["k"].requires_grad_()
        with pytest.raises(Exception, match="no backward"):
            torch.compile(step, backend="eager", fullgraph=True)(*a.values())
