"""GPU: the forms of the attention's kernels that only larger calls choose: 32 rows a wave, and bias windows that are loaded again on the way."""
import pytest
import torch

import seq_ref as R
from test_gpu_seqops import BF16, F16, TYPES, _check_attention, _close, _map, _ops, _pack
from test_gpu_seqops_grads import _dtable

pytestmark = pytest.mark.gpu
HALVES = pytest.mark.parametrize("dtype", [F16, BF16])


def _pairs_of_tiles(lens, kv, group):
    """The forward takes 32 rows a wave from 512 (pairs of sequence and key head times tiles of 128 rows) on."""
    return len(lens) * kv * -(-max(a for a, _ in lens) * group // 128)


@HALVES
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens,heads,kv,dim,nb,span,packed,cut", [
    ([(401, 401)] * 8, 16, 16, 64, 32, 128, False, 0),
    ([(387, 1001)] * 8, 16, 16, 80, 32, 128, False, 0),
    ([(130, 251)] * 9, 48, 16, 64, 16, 64, False, 0),                        # tiles of 126 rows: 42 positions of three heads
    ([(500, 333)] * 8, 32, 16, 128, 0, 0, False, 0),
    ([(200 - 7 * i, 210 - 3 * i) if i not in (3, 9) else (0, i) for i in range(24)], 16, 16, 64, 32, 128, True, 0),
    ([(60 * i % 411, 50 * i % 397) for i in range(16)], 24, 8, 96, 64, 200, True, 37),         # sequences of more rows than max_q are cut
])
def test_attention_with_32_rows_a_wave(dtype, causal, lens, heads, kv, dim, nb, span, packed, cut):
    ops, group = _ops(), heads // kv
    g = torch.Generator().manual_seed(41)
    rows = lambda i, h: [torch.randn(n[i], h, dim, generator=g).to(dtype) for n in lens]  # noqa: E731
    qs, ks, vs = rows(0, heads), rows(1, kv), rows(1, kv)
    table, m = (torch.randn(nb, heads, generator=g), _map(nb, span, not causal)) if nb else (None, None)
    most_q, most_k = max(a for a, _ in lens) - cut, max(b for _, b in lens) - cut
    kw = dict(causal=causal)
    if packed:
        (q, qo), (k, ko), (v, _) = _pack(qs, 2), _pack(ks, 2), _pack(vs, 2)
        kw.update(q_offsets=qo, k_offsets=ko, max_q=most_q, max_k=most_k)
        at = [int(x) for x in qo]
    else:
        q, k, v = (torch.stack(x).cuda() for x in (qs, ks, vs))
    assert _pairs_of_tiles([(min(a, most_q), b) for a, b in lens], kv, group) >= 512
    t, mm = (table.cuda(), m.cuda()) if nb else (None, None)
    out = ops.rel_attention(q, k, v, t, mm, **kw)
    held, saved = ops.rel_attention_train(q, k, v, t, mm, **kw)
    assert torch.equal(out, held)
    if packed:
        owned = torch.zeros(len(q), dtype=torch.bool)
        for i, (a, _) in enumerate(lens):
            owned[at[i]:at[i] + min(a, most_q)] = True
        assert not out[~owned.cuda()].any(), "rows outside every sequence"
    for i in sorted({0, 1, len(lens) // 2, len(lens) - 1}):                  # a sample of the sequences and key heads
        for h in sorted({0, kv - 1}):
            lq, lk = min(lens[i][0], most_q), min(lens[i][1], most_k)
            hs = slice(h * group, (h + 1) * group)
            ref = R.attention(qs[i][:lq, hs], ks[i][:lk, h:h + 1], vs[i][:lk, h:h + 1], table[:, hs] if nb else None, m, dim ** -0.5, causal)
            got = out[at[i]:at[i] + lq, hs] if packed else out[i][:, hs]
            lse = saved.lse[at[i]:at[i] + lq, hs] if packed else saved.lse[i][:, hs]
            _close(got, *ref["out"], f"out of sequence {i}, key head {h}")
            _close(lse, *ref["lse2"], f"lse of sequence {i}, key head {h}")


@TYPES
@pytest.mark.parametrize("lens,heads,kv,dim,causal,nb,span", [
    ((300, 700), 4, 1, 64, True, 64, 600), ((700, 900), 2, 1, 32, False, 32, 1000), ((1200, 1500), 1, 1, 64, False, 64, 1500), ((1100, 1400), 1, 1, 128, True, 256, 2000),
    ((260, 900), 8, 1, 16, True, 16, 700),
])
def test_attention_whose_bias_window_is_loaded_again(dtype, lens, heads, kv, dim, causal, nb, span):
    """Offsets inside the span that a workgroup meets do not fit its window of 2048 / heads offsets: it moves along with the keys (forward, dQ and the table)
    or the rows (dK, dV)."""
    group = heads // kv
    assert min(2 * span, sum(lens)) > 2048 // min(group, 4)
    _check_attention(dtype, [lens], heads, kv, dim, causal, nb, span, packed=False)
    ops = _ops()
    g = torch.Generator().manual_seed(42)
    q, k, v, do = (torch.randn(n, h, dim, generator=g).to(dtype) for n, h in zip((lens[0], lens[1], lens[1], lens[0]), (heads, kv, kv, heads)))
    table, m = torch.randn(nb, heads, generator=g), _map(nb, span, not causal)
    saved = ops.rel_attention_train(q[None].cuda(), k[None].cuda(), v[None].cuda(), table.cuda(), m.cuda(), causal=causal)[1]
    got = ops.rel_attention_grad(saved, do[None].cuda())[3]
    want, square = _dtable(q, k, v, do, table, m, dim ** -0.5, causal)
    # as for the float32 table's gradient in test_gpu_seqops_grads.py; float32 q, k, v multiply with one rounding a product instead of one for 32
    bound = 2.0 ** -19 * square.sqrt()
    off = (got.double().cpu() - want).abs()
    assert bool((off <= 4 * bound + 1e-30).all()) and float(off.norm()) <= float(bound.norm())
