"""CPU: calls of the sequence operators that are refused on the host before anything is planned or launched (made-up addresses are never read)."""
import ctypes as C

import pytest
import torch

from cellvit_amd import _lib, seqops
from test_seqops import A, _attn


@pytest.mark.parametrize("grad", [0, 1])
@pytest.mark.parametrize("heads,kv", [(33, 1), (65, 1), (71, 1), (129, 1), (4096, 2)])
def test_more_than_32_heads_on_a_key_head_are_refused_by_the_workspace_size_too(heads, kv, grad):
    """A tile holds a whole number of positions of a head group: with more than 64 heads none fits, and the plan would divide by 0."""
    for lq, lk in ((1, 20000), (1, 1), (500, 500)):
        a = _attn(heads=heads, kv_heads=kv, max_q=lq, max_k=lk)
        assert _lib.load().cv_op_rel_attention_ws(C.byref(a), grad) == -_lib.CV_ERR_UNSUPPORTED and b"32 query heads" in _lib.load().cv_last_error()


@pytest.mark.parametrize("grad", [0, 1])
@pytest.mark.parametrize("bad,code", [(dict(head_dim=60), 5), (dict(head_dim=0), 5), (dict(head_dim=136), 5), (dict(max_q=1 << 27, heads=32, kv_heads=1), 1), (dict(max_k=1 << 29), 1),
                                      (dict(max_q=-1), 1), (dict(n_seq=1 << 30), 5), (dict(num_buckets=0), 1), (dict(num_buckets=300), 1), (dict(span=-1), 1), (dict(kv_heads=0), 1),
                                      (dict(q_off=A, rows_q=-1), 1), (dict(q_off=A, rows_q=1 << 40), 5), (dict(k_off=A, rows_k=1 << 62), 5), (dict(dtype=2), 1)])
def test_the_workspace_size_refuses_what_the_call_refuses(bad, code, grad):
    a = _attn(**bad)
    assert _lib.load().cv_op_rel_attention_ws(C.byref(a), grad) == -code
    a.ws, a.ws_bytes = A, 1 << 62
    assert getattr(_lib.load(), "cv_op_rel_attention_grad" if grad else "cv_op_rel_attention")(C.byref(a), None) == code


def test_python_raises_what_the_workspace_size_refuses(monkeypatch):
    """Up to the first call into the library nothing needs a GPU."""
    monkeypatch.setattr(seqops, "_same_device", lambda *t: 0)
    q, k = torch.zeros(1, 5, 71, 64), torch.zeros(1, 9, 1, 64)
    for fn in (seqops.rel_attention, seqops.rel_attention_train):
        with pytest.raises(NotImplementedError, match="32 query heads"):
            fn(q, k, k)
    with pytest.raises(NotImplementedError, match="head_dim"):
        seqops.rel_attention(q[:, :, :1, :60], k[..., :60], k[..., :60])
