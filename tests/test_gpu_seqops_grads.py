"""GPU: gradients of the sequence operators held to what their types allow, each entry's errors added as independent ones (the bounds of test_gpu_seqops.py
add the worst of every pair)."""
import ctypes as C
import math

import pytest
import torch

import seq_ref as R
from test_gpu_seqops import BF16, F16, F32, TYPES, _close, _map, _ops, _pack

pytestmark = pytest.mark.gpu
HALVES = pytest.mark.parametrize("dtype", [F16, BF16])


def _dtable(q, k, v, do, table, m, scale, causal):
    """(dtable, sum of squared errors) of one sequence in 64 bits, [buckets, heads].  Everything behind the table's gradient is held in fp32: a score's argument of
    the exponential is below 16 and rounded three times (2^-21 each), so each P is off by less than 2^-19, each on its own; sums of a hundred terms a lane, then
    trees, add 2^-24 sqrt(100) of their size; D = dO . o is off by the same errors of P in the forward.  So an entry is off by 2^-19 times the root of
    the sum over its pairs of (P A)^2, A = |dP| + |D|, and over its rows of (P of the row in the bucket)^2 sum (P dP)^2.  (P rounded to 16 bits in D would put
    2^-9 / sqrt(3) or 2^-11 / sqrt(3) in the place of 2^-19 in the second.)"""
    q, k, v, do, t = (x.cpu().double() for x in (q, k, v, do, table))
    (lq, H, _), (lk, Hk, _) = q.shape, k.shape
    nb = t.shape[0]
    value, square = torch.zeros(nb, H, dtype=torch.float64), torch.zeros(nb, H, dtype=torch.float64)
    if lq == 0 or lk == 0:
        return value, square
    plane = R.bucket_plane(m, lq, lk)
    flat = plane.reshape(-1)
    for h in range(H):
        g = h // (H // Hk)
        s = scale * q[:, h] @ k[:, g].T + t[:, h][plane]
        if causal:
            s = s.masked_fill(torch.arange(lk)[None] > torch.arange(lq)[:, None] + lk - lq, -math.inf)
        lse = torch.logsumexp(s, 1, keepdim=True)
        p = torch.where(lse == -math.inf, torch.zeros(()).double(), torch.exp(s - lse.clamp(min=-1e300)))
        dp = do[:, h] @ v[:, g].T
        d = (p * dp).sum(1, keepdim=True)
        value[:, h].index_add_(0, flat, (p * (dp - d)).reshape(-1))
        square[:, h].index_add_(0, flat, (p * (dp.abs() + d.abs())).square().reshape(-1))
        mass = torch.zeros(lq, nb, dtype=torch.float64).scatter_add_(1, plane, p)
        square[:, h] += (mass.square() * (p * dp).square().sum(1, keepdim=True)).sum(0)
    return value, square


@HALVES
@pytest.mark.parametrize("lens,heads,kv,dim,causal,nb,span,packed", [
    ([(257, 257)] * 2, 3, 3, 64, False, 32, 128, False),
    ([(700, 700)], 2, 2, 64, False, 32, 128, False),
    ([(300, 411)], 4, 2, 128, True, 64, 200, False),
    ([(3, 700)], 4, 2, 80, True, 32, 64, False),                             # few rows: the keys are split and the parts joined
    ([(5, 40)], 2, 1, 128, False, 16, 20, False),                            # few rows, one part
    ([(20, 1500)], 1, 1, 32, False, 32, 128, False),                         # more rows, split keys
    ([(130, 130), (0, 0), (7, 90), (1, 1), (200, 64)], 6, 6, 64, True, 32, 128, True),
    ([(400, 400)] * 8, 16, 16, 32, False, 32, 128, False),                   # 32 rows a wave
    ([(390, 390)] * 8, 16, 16, 128, True, 32, 300, False),
    ([(260, 260)] * 3, 126, 42, 96, False, 16, 64, False),                   # 32 rows a wave, tiles of 126 rows
])
def test_a_float32_tables_gradient_is_good_to_float32(dtype, lens, heads, kv, dim, causal, nb, span, packed):
    ops = _ops()
    g = torch.Generator().manual_seed(31)
    rows = lambda i, h: [torch.randn(n[i], h, dim, generator=g).to(dtype) for n in lens]  # noqa: E731
    qs, ks, vs, dos = rows(0, heads), rows(1, kv), rows(1, kv), rows(0, heads)
    table, m = torch.randn(nb, heads, generator=g), _map(nb, span, not causal)
    kw = dict(causal=causal)
    if packed:
        (q, qo), (k, ko) = _pack(qs, 2), _pack(ks, 2)
        v, do = _pack(vs, 2)[0], _pack(dos, 2)[0]
        kw.update(q_offsets=qo, k_offsets=ko, max_q=max(a for a, _ in lens), max_k=max(b for _, b in lens))
    else:
        q, k, v, do = (torch.stack(x).cuda() for x in (qs, ks, vs, dos))
    out, saved = ops.rel_attention_train(q, k, v, table.cuda(), m.cuda(), **kw)
    with torch.no_grad():
        assert torch.equal(out, ops.rel_attention(q, k, v, table.cuda(), m.cuda(), **kw))
    got = ops.rel_attention_grad(saved, do)[3]
    assert got.dtype == torch.float32
    parts = [_dtable(a, b, c, d, table, m, dim ** -0.5, causal) for a, b, c, d in zip(qs, ks, vs, dos)]
    want, bound = sum(p[0] for p in parts), 2.0 ** -19 * sum(p[1] for p in parts).sqrt()
    off = (got.double().cpu() - want).abs()
    # an entry's error is a sum of independent ones: four times its size is allowed, once for their norm
    assert bool((off <= 4 * bound + 1e-30).all()), f"worst {float((off / bound.clamp(min=1e-30)).max()):.1f} x its size"
    assert float(off.norm()) <= float(bound.norm())


@HALVES
@pytest.mark.parametrize("junk", [math.nan, math.inf, 65504.0, -1e4])
def test_what_cut_and_unowned_rows_hold_changes_no_gradient(dtype, junk):
    """Sequences longer than max_q / max_k are cut there: the rest belongs to no sequence, nor do the rows before the first and behind the last."""
    ops = _ops()
    g = torch.Generator().manual_seed(32)
    mk = lambda n: torch.randn(n, 2, 64, generator=g).to(dtype)  # noqa: E731
    q, k, v, do = mk(230), mk(260), mk(260), mk(230)
    qo, ko = torch.tensor([5, 105, 105, 225], dtype=torch.int32), torch.tensor([3, 123, 133, 255], dtype=torch.int32)
    table, m = torch.randn(16, 2, generator=g).cuda(), _map(16, 20, True).cuda()
    lost_q, lost_k = torch.ones(230, dtype=torch.bool), torch.ones(260, dtype=torch.bool)
    for a, b in zip(qo[:-1].tolist(), qo[1:].tolist()):
        lost_q[a:min(b, a + 70)] = False
    for a, b in zip(ko[:-1].tolist(), ko[1:].tolist()):
        lost_k[a:min(b, a + 90)] = False
    res = []
    for fill in (0.0, junk):
        a, b, c, d = (t.clone() for t in (q, k, v, do))
        for t, lost in ((a, lost_q), (b, lost_k), (c, lost_k), (d, lost_q)):
            t[lost] = fill
        out, saved = ops.rel_attention_train(a.cuda(), b.cuda(), c.cuda(), table, m, q_offsets=qo.cuda(), k_offsets=ko.cuda(), max_q=70, max_k=90)
        res.append([out, *ops.rel_attention_grad(saved, d.cuda())])
    for x, y in zip(*res):
        assert bool(torch.isfinite(y).all()) and torch.equal(x, y)


@HALVES
@pytest.mark.parametrize("dscale,vscale,dim", [(0.01, 8000.0, 128), (0.02, 60000.0, 64), (100.0, 2.0, 64), (3e-5, 1.0, 64), (1.0, 1e-3, 32)])
def test_gradients_that_fit_their_type_survive_large_and_small_values(dtype, dscale, vscale, dim):
    """dout and v of one sign pattern, two keys: |dP| is dim dscale vscale, the largest there can be for these sizes, and |dS| up to half of it."""
    ops = _ops()
    g = torch.Generator().manual_seed(33)
    lq, lk = 6, 2
    pattern = torch.randn(dim, generator=g).sign()
    side = torch.tensor([1.0, -1.0]).view(lk, 1, 1)
    q, k = (torch.randn(1, n, 1, dim, generator=g).to(dtype) for n in (lq, lk))
    k = (k.float() * 0.1).to(dtype)
    v = (pattern * side * vscale).to(dtype)[None]
    do = (pattern.expand(1, lq, 1, dim) * dscale).to(dtype)
    ref = R.attention(q[0], k[0], v[0], None, None, dim ** -0.5, False, do[0])
    saved = ops.rel_attention_train(q.cuda(), k.cuda(), v.cuda())[1]
    got = ops.rel_attention_grad(saved, do.cuda())
    for name, x in zip(("dq", "dk", "dv"), got):
        want, bound = ref[name]
        assert bool(torch.isfinite(want.to(dtype)).all()) and bool(torch.isfinite(x).all()), name
        assert bool(((x[0].double().cpu() - want).abs() <= bound).all()), name


def _rounded_once(want, dtype, terms):
    """Size of the error of a result that is rounded once and sums rounded dS: `terms` is the root of the sum of squares of what it sums, each rounded by
    u / sqrt(3) of itself (independent; fp16's own subnormals are in the result's rounding)."""
    return math.hypot(float((want.to(dtype).double() - want).norm()), R.half_step(dtype) / math.sqrt(3) * float(terms.norm()))


def _root_of_squares(q, k, v, do, causal):
    """One head: dq, dk in 64 bits and, for each element, the root of the sum of the squares of its terms."""
    q, k, v, do = (x[:, 0].double() for x in (q, k, v, do))
    s = q @ k.T * q.shape[1] ** -0.5
    if causal:
        s = s.masked_fill(torch.arange(len(k))[None] > torch.arange(len(q))[:, None] + len(k) - len(q), -math.inf)
    p, dp = s.softmax(-1), do @ v.T
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * q.shape[1] ** -0.5
    return ds @ k, ds.T @ q, (ds.square() @ k.square()).sqrt(), (ds.square().T @ q.square()).sqrt()


@HALVES
@pytest.mark.parametrize("sizes", [(300.0, 3.0, 0.03), (0.03, 300.0, 3.0), (1.0, 1e-2, 1e2)])
def test_a_sequences_gradients_do_not_hang_on_its_neighbours(dtype, sizes):
    """Sequences of one call whose dout differ by 1e2 to 1e4, as a loss that is a mean over each sequence's tokens makes them."""
    ops = _ops()
    g = torch.Generator().manual_seed(34)
    lens, dim = (700, 333, 1500), 64
    mk = lambda n, by=1.0: (torch.randn(n, 1, dim, generator=g) * by).to(dtype)  # noqa: E731
    parts = [(mk(n), mk(n), mk(n), mk(n, by)) for n, by in zip(lens, sizes)]
    off = torch.tensor([0, *torch.tensor(lens).cumsum(0).tolist()], dtype=torch.int32).cuda()
    q, k, v, do = (torch.cat(x).cuda() for x in zip(*parts))
    saved = ops.rel_attention_train(q, k, v, q_offsets=off, k_offsets=off, max_q=1500, max_k=1500)[1]
    got = ops.rel_attention_grad(saved, do)
    at = 0
    for n, part in zip(lens, parts):
        dq, dk, tq, tk = _root_of_squares(*part, False)
        for name, x, want, terms in (("dq", got[0], dq, tq), ("dk", got[1], dk, tk)):
            off_by = float((x[at:at + n, 0].double().cpu() - want).norm())
            # of independent errors: their norm strays by 1 / sqrt(2 n), 5 % are allowed for their not being uniform
            assert off_by <= 1.05 * _rounded_once(want, dtype, terms), (name, n, off_by / _rounded_once(want, dtype, terms))
        at += n


@HALVES
def test_gradients_of_rows_and_keys_hang_on_their_own_dout(dtype):
    """Causal, the rows' dout falling by 1e4 along the sequence: the last keys are seen by small rows only."""
    ops = _ops()
    g = torch.Generator().manual_seed(35)
    n, dim = 1024, 64
    by = 10.0 ** torch.linspace(1.5, -2.5, 8)
    q, k, v, do = (torch.randn(n, 1, dim, generator=g).to(dtype) for _ in range(4))
    k, q = (k.float() * 2).to(dtype), (q.float() * 2).to(dtype)
    do = (do.float() * by.repeat_interleave(n // 8)[:, None, None]).to(dtype)
    saved = ops.rel_attention_train(q[None].cuda(), k[None].cuda(), v[None].cuda(), causal=True)[1]
    got = ops.rel_attention_grad(saved, do[None].cuda())
    dq, dk, tq, tk = _root_of_squares(q, k, v, do, True)
    for name, x, want, terms in (("dq", got[0], dq, tq), ("dk", got[1], dk, tk)):
        for i in range(8):
            part = slice(i * n // 8, (i + 1) * n // 8)
            off_by = float((x[0, part, 0].double().cpu() - want[part]).norm())
            assert off_by <= 1.05 * _rounded_once(want[part], dtype, terms[part]), (name, i, off_by / _rounded_once(want[part], dtype, terms[part]))


@HALVES
@pytest.mark.parametrize("lk,dim", [(4096, 128), (32768, 64), (131072, 64)])
def test_gradients_of_values_among_many_keys(dtype, lk, dim):
    ops = _ops()
    g = torch.Generator().manual_seed(36)
    lq = 48
    q, k, v, do = (torch.randn(n, 1, dim, generator=g).to(dtype) for n in (lq, lk, lk, lq))
    do = (do.float() * lk / 64).to(dtype)                                    # gradients of normal size
    saved = ops.rel_attention_train(q[None].cuda(), k[None].cuda(), v[None].cuda())[1]
    got = ops.rel_attention_grad(saved, do[None].cuda())[2][0, :, 0].double().cpu()
    qd, kd, dd = (x[:, 0].double() for x in (q, k, do))
    p = (qd @ kd.T * dim ** -0.5).softmax(-1)
    want, terms = p.T @ dd, (p.T.square() @ dd.square()).sqrt()
    off_by, size = float((got - want).norm()), _rounded_once(want, dtype, terms)
    assert off_by <= 1.05 * size, off_by / size


@TYPES
def test_rows_of_no_sequence_are_zeroed_where_there_is_nothing_to_attend_to(dtype):
    """No sequences, or none of any length: packed rows belong to nobody and get zeros from the C entries, too (zero_rest), or stay as they were."""
    from cellvit_amd import _lib
    lib, code = _lib.load(), {F16: _lib.DTYPE_F16, BF16: _lib.DTYPE_BF16, F32: _lib.DTYPE_F32}[dtype]
    T, H, D = 37, 3, 24
    for n_seq, most_q, most_k in ((0, 5, 5), (2, 0, 5), (2, 5, 0)):
        off = torch.full((n_seq + 1,), 10, dtype=torch.int32, device="cuda")
        q, do = (torch.randn(T, H, D, device="cuda").to(dtype) for _ in range(2))
        for zero in (0, 1):
            out = torch.full((T, 2 * H, D), 7.0, dtype=dtype, device="cuda")[:, H:]           # strided: every second block of heads
            grads = [torch.full((T, H, D), 7.0, dtype=dtype, device="cuda") for _ in range(3)]
            lse, ws = torch.zeros(T, H, device="cuda"), torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
            a = _lib.cv_rel_attn(dtype=code, n_seq=n_seq, heads=H, kv_heads=H, head_dim=D, max_q=most_q, max_k=most_k, scale=0.2, zero_rest=zero, rows_q=T, rows_k=T, q_row=H * D,
                                 q_head=D, k_row=H * D, k_head=D, v_row=H * D, v_head=D, o_row=2 * H * D, o_head=D, do_row=H * D, do_head=D, q=q.data_ptr(), k=q.data_ptr(),
                                 v=q.data_ptr(), q_off=off.data_ptr(), k_off=off.data_ptr(), out=out.data_ptr(), lse=lse.data_ptr(), dout=do.data_ptr(), dq=grads[0].data_ptr(),
                                 dk=grads[1].data_ptr(), dv=grads[2].data_ptr(), ws=ws.data_ptr(), ws_bytes=ws.numel())
            for fn in (lib.cv_op_rel_attention, lib.cv_op_rel_attention_grad):
                _lib.check(fn(C.byref(a), torch.cuda.current_stream().cuda_stream))
            want = 0.0 if zero else 7.0
            for t in (out, *grads):
                assert bool((t == want).all()), (n_seq, most_q, most_k, zero)
            assert bool((out._base[:, :H] == 7).all())
        got = _ops().rel_attention(q, q, q, q_offsets=off, k_offsets=off, max_q=most_q, max_k=most_k)
        assert not got.any()


@TYPES
@pytest.mark.parametrize("packed_q", [False, True])
def test_one_side_packed_and_the_other_dense(dtype, packed_q):
    """Single tokens or a few rows a sequence beside packed keys of any length, and the other way round."""
    ops = _ops()
    g = torch.Generator().manual_seed(37)
    long, short = [0, 1, 700, 63], 3
    lq, lk = (long, [short] * 4) if packed_q else ([short] * 4, long)
    mk = lambda n, h: [torch.randn(x, h, 64, generator=g).to(dtype) for x in n]  # noqa: E731
    qs, ks, vs, dos = mk(lq, 4), mk(lk, 2), mk(lk, 2), mk(lq, 4)
    table, m = torch.randn(16, 4, generator=g), _map(16, 20, True)
    off = torch.tensor([0, *torch.tensor(long).cumsum(0).tolist()])                            # 64-bit offsets are taken, too
    join = lambda x, packed: (torch.cat if packed else torch.stack)(x).cuda()  # noqa: E731
    kw = dict(q_offsets=off.cuda(), max_q=700) if packed_q else dict(k_offsets=off.cuda(), max_k=700)
    q, do, k, v = join(qs, packed_q), join(dos, packed_q), join(ks, not packed_q), join(vs, not packed_q)
    out, saved = ops.rel_attention_train(q, k, v, table.cuda(), m.cuda(), **kw)
    assert torch.equal(out, ops.rel_attention(q, k, v, table.cuda(), m.cuda(), **kw))
    dq, dk, dv, dt = ops.rel_attention_grad(saved, do)
    part = lambda x, i, packed: x[off[i]:off[i + 1]] if packed else x[i]  # noqa: E731
    refs = [R.attention(*x, table, m, 0.125, False, d) for *x, d in zip(qs, ks, vs, dos)]
    for i, r in enumerate(refs):
        for name, x, p in (("out", out, packed_q), ("dq", dq, packed_q), ("dk", dk, not packed_q), ("dv", dv, not packed_q)):
            _close(part(x, i, p), *r[name], name)
    _close(dt, sum(r["dtable"][0] for r in refs), sum(r["dtable"][1] for r in refs), "dtable")


@HALVES
@pytest.mark.parametrize("lens,heads,kv,dim", [((2, 600), 16, 2, 128), ((90, 90), 32, 1, 128), ((150, 700), 6, 2, 80)])
def test_training_halves_whose_first_call_is_captured(dtype, lens, heads, kv, dim):
    """Kernels that ask for more than 64 KB of LDS, workspaces and all, inside a capture; replays with other inputs and eager work between."""
    ops = _ops()
    g = torch.Generator().manual_seed(38)
    fresh = lambda: [torch.randn(1, n, h, dim, generator=g).to(dtype).cuda() for n, h in zip((lens[0], lens[1], lens[1], lens[0]), (heads, kv, kv, heads))]  # noqa: E731
    table, m = torch.randn(256, heads, generator=g).cuda(), _map(256, 300, False).cuda()

    def step(q, k, v, do):
        out, saved = ops.rel_attention_train(q, k, v, table, m, causal=True)
        return [out, saved.lse, saved.out_lo, *ops.rel_attention_grad(saved, do)]
    state = fresh()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(*state)
    for scale in (1.0, 1e-3, 300.0):
        new = fresh()
        new[3] *= scale
        for a, b in zip(state, new):
            a.copy_(b)
        graph.replay()
        got = [t.clone() for t in held]
        want = step(*new)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@HALVES
def test_autograd_with_a_float32_table_equals_the_halves(dtype):
    ops = _ops()
    g = torch.Generator().manual_seed(39)
    q, k, v = (torch.randn(2, 130, 3, 64, generator=g).to(dtype).cuda().requires_grad_(True) for _ in range(3))
    table, m = torch.randn(3, 32, generator=g).cuda().T.requires_grad_(True), _map(32, 50, True).cuda()      # [buckets, heads], not contiguous
    do = torch.randn(2, 130, 3, 64, generator=g).to(dtype).cuda()
    out = ops.rel_attention(q, k, v, table, m)
    got = torch.autograd.grad(out, (q, k, v, table), do)
    want = ops.rel_attention_grad(ops.rel_attention_train(*(t.detach() for t in (q, k, v, table)), m)[1], do)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[3].dtype == torch.float32
    same = torch.autograd.grad(ops.rel_attention(q, q, q, table, m), q, do)[0]                 # one tensor in three places
    parts = ops.rel_attention_grad(ops.rel_attention_train(q.detach(), q.detach(), q.detach(), table.detach(), m)[1], do)[:3]
    total = sum(t.double() for t in parts)
    assert float((same.double() - total).norm()) <= 3 * R.half_step(dtype) * float(sum(t.double().abs() for t in parts).norm())


@TYPES
@pytest.mark.parametrize("lens", [(150, 170), (2, 900)])
def test_the_c_entries_take_any_form_of_what_rounding_took(dtype, lens):
    """out_lo in fp32, in the call's type, or none: the same output, and gradients as good as D allows."""
    from cellvit_amd import _lib
    lib, code = _lib.load(), {F16: _lib.DTYPE_F16, BF16: _lib.DTYPE_BF16, F32: _lib.DTYPE_F32}[dtype]
    g = torch.Generator().manual_seed(40)
    (lq, lk), H, D = lens, 2, 64
    q, k, v, do = (torch.randn(n, H, D, generator=g).to(dtype) for n in (lq, lk, lk, lq))
    table, m = torch.randn(32, H, generator=g), _map(32, 64, True)
    dev = [t.cuda() for t in (q, k, v, do, table, m)]
    ref = R.attention(q, k, v, table, m, 0.125, False, do)
    off, outs = [], []
    for lo in (torch.full((lq, H, D), 7.0, device="cuda"), torch.full((lq, H, D), 7.0, dtype=dtype, device="cuda"), None):
        out, dq, dk, dv = (torch.empty(n, H, D, dtype=dtype, device="cuda") for n in (lq, lq, lk, lk))
        lse, dt = torch.empty(lq, H, device="cuda"), torch.empty(32, H, device="cuda")
        a = _lib.cv_rel_attn(dtype=code, n_seq=1, heads=H, kv_heads=H, head_dim=D, max_q=lq, max_k=lk, num_buckets=32, span=64, scale=0.125, table_dtype=_lib.DTYPE_F32,
                             lo_f32=int(lo is not None and lo.dtype is F32), q_row=H * D, q_head=D, k_row=H * D, k_head=D, v_row=H * D, v_head=D, o_row=H * D, o_head=D, do_row=H * D, do_head=D,
                             q=dev[0].data_ptr(), k=dev[1].data_ptr(), v=dev[2].data_ptr(), table=dev[4].data_ptr(), map=dev[5].data_ptr(), out=out.data_ptr(), lse=lse.data_ptr(),
                             out_lo=None if lo is None else lo.data_ptr(), dout=dev[3].data_ptr(), dq=dq.data_ptr(), dk=dk.data_ptr(), dv=dv.data_ptr(), dtable=dt.data_ptr())
        for grad, fn in enumerate((lib.cv_op_rel_attention, lib.cv_op_rel_attention_grad)):
            need = lib.cv_op_rel_attention_ws(C.byref(a), grad)
            ws = torch.empty(max(need, 16), dtype=torch.uint8, device="cuda")
            a.ws, a.ws_bytes = ws.data_ptr(), need
            _lib.check(fn(C.byref(a), torch.cuda.current_stream().cuda_stream))
            torch.cuda.synchronize()
        for name, x in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv), ("dtable", dt)):
            _close(x, *ref[name], name)
        outs.append(out)
        off.append(float((dt.double().cpu() - ref["dtable"][0]).norm() / ref["dtable"][0].norm()))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    if dtype != F32:                                                         # D good to fp32, to about 16 bits more than `dtype`, to `dtype`
        assert off[0] <= 2.0 ** -17 and off[1] <= 2.0 ** -14 and off[0] <= off[2] and off[1] <= off[2]


@TYPES
@pytest.mark.parametrize("batch,heads,q,k", [(64, 2, 257, 257), (512, 1, 130, 131), (3, 2, 1000, 700)])
def test_a_planes_gradient_summed_over_a_batch_of_one_sign(dtype, batch, heads, q, k):
    """Values near 0.1: every addition to a running sum errs the same way.  A lane adds runs of 128 rows, the batch's runs with compensation (2^-23 in all), and the
    diagonals and parts in trees of some 30 additions: (128 + 30) 2^-24 of the sum at the worst."""
    ops = _ops()
    g = torch.Generator().manual_seed(43)
    d = (0.1 + 0.001 * torch.rand(batch, heads, q, k, generator=g)).to(dtype)
    m = _map(32, 128, True)
    got = ops.rel_bias_grad(d.cuda(), m.cuda(), 32).double().cpu()
    plane, total = R.bucket_plane(m, q, k).reshape(-1), d.double().sum(0).reshape(heads, -1)
    want = torch.zeros(32, heads, dtype=torch.float64).index_add_(0, plane, total.T)
    assert float(((got - want).abs() / want.abs().clamp(min=1e-30)).max()) <= 160 * 2.0 ** -24


@TYPES
def test_logarithms_of_the_sums_err_to_both_sides(dtype):
    """lse is near 8 .. 12, where a step is 2^-20: rounded once, to both sides alike; the logarithm of 1/2 .. 1 and the exponentials may lean by a step of 2^-24 each."""
    ops = _ops()
    g = torch.Generator().manual_seed(44)
    q, k = (torch.randn(1, 1500, 2, 64, generator=g).to(dtype) for _ in range(2))
    lse = ops.rel_attention_train(q.cuda(), k.cuda(), k.cuda())[1].lse.double().cpu()[0]
    s = q[0].double().transpose(0, 1) @ k[0].double().permute(1, 2, 0) * 0.125
    off = lse - torch.logsumexp(s, 2).T / math.log(2)
    assert float(off.abs().max()) <= 2.0 ** -19 and abs(float(off.mean())) <= 2.0 ** -23
