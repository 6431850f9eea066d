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


@pytest.mark.parametrize("grad", [False, True])
def test_tensors_that_carry_a_forward_mode_tangent_are_refused(grad):
    """The kernels would return a tensor without one, as if the derivative were zero."""
    import torch.autograd.forward_ad as fwd
    t = torch.zeros
    m = seqops.rel_buckets(8, 16, True, device="cpu")
    q, table, x, w = t(1, 5, 2, 16), t(8, 2), t(6, 32), t(32)
    saved = seqops.RelAttentionSaved(q, q, q, table, m, None, None, q, t(1, 5, 2), None, 0.25, False, 5, 5)
    kept = seqops.BlockNormSaved(x, x, t(6, 4), None, (w, None), None, 6, 1.0, "layer", 1e-6)
    with fwd.dual_level():
        d = lambda p: fwd.make_dual(p.clone().requires_grad_(grad), torch.ones_like(p))  # noqa: E731
        calls = [lambda: seqops.rel_bias(d(table), m, 3, 3), lambda: seqops.rel_bias_grad(d(t(2, 3, 3)), m, 8), lambda: seqops.rel_attention(d(q), q, q),
                 lambda: seqops.rel_attention(q, q, d(q)), lambda: seqops.rel_attention(q, q, q, d(table), m), lambda: seqops.rel_attention_train(q, d(q), q),
                 lambda: seqops.rel_attention_grad(saved, d(q)), lambda: seqops.rel_attention_grad(saved._replace(v=d(q)), q), lambda: seqops.block_norm(d(x), x, pre=w),
                 lambda: seqops.block_norm(x, d(x), pre=w), lambda: seqops.block_norm(x, x, post=(w, d(w))), lambda: seqops.block_norm(x, x, gate=d(w)),
                 lambda: seqops.block_norm_train(x, x, pre=d(w)), lambda: seqops.block_norm_grad(kept, d(x), None), lambda: seqops.block_norm_grad(kept, x, d(x))]
        for call in calls:
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                call()
        with pytest.raises(RuntimeError, match="no CPU fallback"):                             # a level alone changes nothing
            seqops.rel_attention(q, q, q)


def test_sizes_beyond_32_bits_are_refused_and_wide_gate_groups_are_one_group(monkeypatch):
    """None of them may reach the library with its upper bits cut off."""
    t = torch.zeros
    m = seqops.rel_buckets(8, 16, True, device="cpu")
    monkeypatch.setattr(seqops, "_same_device", lambda *a: 0)
    calls = []
    monkeypatch.setattr(seqops, "_call", lambda device, fn, a, *rest: calls.append(a))
    q, off, x = t(7, 2, 16), torch.tensor([0, 7], dtype=torch.int32), t(6, 32)
    for lq, lk in ((1 << 31, 7), (7, 1 << 40), (-1 << 40, 7), ((1 << 32) + 7, 7)):
        with pytest.raises(ValueError):
            seqops.rel_attention(q, q, q, q_offsets=off, k_offsets=off, max_q=lq, max_k=lk)
    for lq, lk in (((1 << 32) + 3, 3), (3, (1 << 32) + 3), (-1, 3), (3, 1 << 23)):
        with pytest.raises(ValueError):
            seqops.rel_bias(t(8, 2), m, lq, lk)
    for nb in (0, 257, (1 << 32) + 8):
        with pytest.raises(ValueError):
            seqops.rel_bias_grad(t(2, 3, 3), m, nb)
    with pytest.raises(NotImplementedError):
        seqops.rel_attention(q[:1].expand(1 << 31, 2, 16), q, q, q_offsets=off, k_offsets=off, max_q=7, max_k=7)
    with pytest.raises(ValueError):
        seqops.block_norm(x, x, gate=t(2, 32), rows_per_gate=1 << 40)      # one group, not two
    assert not calls
    for per in (6, 7, 1 << 31, 1 << 40):
        seqops.block_norm(x, x, gate=t(1, 32), rows_per_gate=per)
    assert len(calls) == 4 and len({a[:24] for a in calls}) == 1               # the head of the struct: sizes and rows a group


def test_what_rounding_took_must_be_float32():
    t = torch.zeros
    q = t(1, 5, 2, 16).half()
    saved = seqops.RelAttentionSaved(q, q, q, None, None, None, None, q, t(1, 5, 2), t(1, 5, 2, 16), 0.25, False, 5, 5)
    for bad in (q, t(1, 5, 2, 8), t(1, 5, 16, 2).transpose(2, 3)):
        with pytest.raises(ValueError, match="out_lo"):
            seqops.rel_attention_grad(saved._replace(out_lo=bad), q)
