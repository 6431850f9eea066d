// Attention with a bucketed position bias, backward:
//   P = 2^(s - lse),  dV = P^T dO,  dP = dO V^T,  dS = P (dP - D),  D_i = dO_i . o_i,  dQ = scale dS K,  dK = scale dS^T Q,  dt[c] = sum dS over bucket c
// Two kernels that each own what they write (dQ and the table's gradient by rows, dK and dV by keys), so no sum depends on scheduling; the price is
// seven products where five would do.
// fp16: a row's dS is scaled by a power of two from |dO_i| and max |V_j| for the products (exact, taken out of the results): ds_exponent.
#include <initializer_list>

#include "relattn.h"

namespace cva {
namespace {

// fp16: the largest |V_j|^2 of a (sequence, key head) pair, in n_amax parts.  Rows that no sequence owns, those it was cut by among them, hold anything and are
// left out.  16 lanes a row.
template <typename T>
__global__ __launch_bounds__(256) void rel_vnorm_kernel(const RelAttn k) {
    __shared__ float red[4];
    const cv_rel_attn& a = k.a;
    const int c = (threadIdx.x & 15) * 8, D = a.head_dim, pair = (int)blockIdx.x / k.n_amax, part = (int)blockIdx.x - pair * k.n_amax;
    const int s = pair / a.kv_heads, kvh = pair - s * a.kv_heads;
    const SeqRange kr = seq_range(a.k_off, s, a.max_k, a.rows_k);
    const T* vb = reinterpret_cast<const T*>(a.v) + (a.k_off ? kr.row0 * a.v_row : s * a.v_seq) + (long)kvh * a.v_head;
    float top = 0.f;
    for (int r0 = part * 16; r0 < kr.len; r0 += k.n_amax * 16) {
        const int r = r0 + ((int)threadIdx.x >> 4);
        const v8<T> d = frag_global(vb + (long)r * a.v_row, c, D, r < kr.len);
        float n = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) n = fmaf((float)d[j], (float)d[j], n);
#pragma unroll
        for (int x = 8; x; x >>= 1) n += __shfl_xor(n, x);
        top = fmaxf(top, n);
    }
#pragma unroll
    for (int x = 32; x >= 16; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) k.amax[blockIdx.x] = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

// Exponent e of the factor 2^e on the dS of a row, b2 = |dO_i|^2 max |V_j|^2: |dP| <= B = sqrt(b2), so |dS| = P |dP - D| <= B / 2 (the other pairs' mean is at most
// 2 B away and P (1 - P) <= 1/4); B 2^e lies in 2^14 .. 2^15, so nothing that fits fp16 overflows, and 2^28 lie between the largest dS and the
// subnormals.  Each row of dQ has its own; dK takes the smallest of the rows its keys meet, tile by tile.
constexpr int DS_FREE = 64;                                                  // a row of dS = 0
__device__ __forceinline__ int ds_exponent(float b2) {
    if (!(b2 > 0.f)) return DS_FREE;
    return 14 - (((int)(__float_as_uint(b2) >> 23) - 127) >> 1);             // -50 for infinities
}
template <typename T> constexpr bool SCALED = __is_same(T, half_t);
// fp16's P for dV rides on 2^14: P <= 1, and beside 1e5 keys most of it would be subnormal (1.4e-3 of dV at 131072 keys).  It is added to the exponent.
template <typename T> constexpr int P_UP = SCALED<T> ? 14 : 0;
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((unsigned)(127 + e) << 23); }

// waves a SIMD to leave registers for: fp32 fragments of wide heads need more than half of them
template <typename T> constexpr int grad_waves(int DT) { return sizeof(T) == 4 && DT > 80 ? 1 : 2; }

// the smaller of v and, where the row mask takes part, what CTRL brings from another lane
template <int CTRL, int ROWS> __device__ __forceinline__ int dpp_min(int v) {
    const int w = __builtin_amdgcn_update_dpp(v, v, CTRL, ROWS, 0xf, false);
    return w < v ? w : v;
}
template <int CTRL> __device__ __forceinline__ float dpp_shift(float v) {
    return __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xf, 0xf, true));
}

// dQ and the table's gradient.  S^T and dP^T [key][query], dQ^T += K^T dS^T.  A tile holds k.qt positions (a multiple of 16) of k.ht heads that share the key
// head, head by head: every block of 16 rows is 16 neighbouring positions of one head.
// Table: all pairs of a diagonal (key minus position) share a bucket.  In a 16 x 16 block of dS^T lane (g4, x) holds rows 4 g4 + r of column x, diagonal
// 4 g4 + r - x: shifting register r by r lanes brings diagonal 4 g4 - x of a lane group together in lane x (3 additions); what leaves the row at
// its lower end, diagonals 4 g4 + 1 .. 3, is lanes 13 .. 15 of the next block of keys, where it is carried to.  So a lane's sum of a block belongs to one
// offset, 16 further a block, and to one bucket for many blocks: it stays in a register until some lane's bucket changes.  Where one bucket ends, its
// lanes' sums are added over the wave; where several do (near the diagonal) the wave's sums are put in the order of their offsets through LDS
// and added by bucket.  (Causal step of 2 x 16 heads x 4096 x 128, right after a pause: 486 us, 446 with the case of one bucket by itself, 363 without table;
// 400 in a run of steps.  Adding every block's sums to LDS by atomics cost 100 cycles an instruction, 60 % of the kernel.)  A tile beyond the span adds to
// one sum a lane.
// Bound by issue: of 24 products' 384 cycles a tile and wave a third runs at once with the loads, exponentials and sums of the other waves.
// Closer to the diagonal than ZONE the sums are kept by offset, and added by bucket at the end: buckets are narrow there (ragged step of 24 x 12 heads x
// 64, span 128: 518 us without, 506; 516 with 48 or 240, whose LDS and last sums cost what they save).
constexpr int ZONE = 112, WAVE_SUMS = 160 + 2 * ZONE + 32;
template <typename T, int DT, int BK>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? (DT <= 64 ? 4 : DT <= 96 ? 3 : 2) : grad_waves<T>(DT)) void rel_attn_dq_kernel(const RelAttn k) {
    typedef Dims<DT> Dm;
    constexpr int NB = BK / 16, PT = pitch_of<T>(Dm::W);
    extern __shared__ __attribute__((aligned(32))) char lds[];
    const cv_rel_attn& a = k.a;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g4 = lane >> 4, li = lane & 15;
    const int nb = a.num_buckets;
    T* tiles = reinterpret_cast<T*>(lds);                                    // K, V; K, V
    float* tab = reinterpret_cast<float*>(tiles + 4 * BK * PT);
    float* window = tab + k.ht * nb;
    uint8_t* bwin = reinterpret_cast<uint8_t*>(window + k.ht * k.win);       // buckets of the window's offsets
    float* order = window + k.ht * k.win + k.win / 4 + wave * WAVE_SUMS;     // [4][32] sums, [32] buckets by offset
    float* diag = order + 160;                                               // sums of the offsets -ZONE - 15 .. ZONE + 16
    float* bacc = window + k.ht * k.win + k.win / 4 + 4 * WAVE_SUMS + wave * nb;           // this wave's bucket sums

    Part me;
    if (!part_of_block(k, me)) return;
    const int tile = me.tile, kvh = me.kvh, s = me.s;
    if (a.q_off && a.zero_rest && tile + kvh == 0)
        zero_rest(a.q_off, s, a.n_seq, a.max_q, a.rows_q, reinterpret_cast<T*>(a.dq), (long)a.heads * a.head_dim, a.heads, a.head_dim, a.head_dim);
    const int hsplit = (k.G + k.ht - 1) / k.ht, h0 = tile % hsplit * k.ht;
    int ptile = tile / hsplit;
    const int ptiles = k.tiles / hsplit;
    if (a.causal) ptile = ptiles - 1 - ptile;
    const SeqRange qr = seq_range(a.q_off, s, a.max_q, a.rows_q), kr = seq_range(a.k_off, s, a.max_k, a.rows_k);
    const int q0 = ptile * k.qt, shift = kr.len - qr.len, D = a.head_dim, nh = k.G - h0 < k.ht ? k.G - h0 : k.ht;
    const int qn = qr.len - q0 < k.qt ? qr.len - q0 : k.qt;                  // positions of this tile
    const int blocks = k.qt / 16;                                            // of one head
    const int blk = wave % blocks, head = wave / blocks;
    const bool on = head < nh && blk * 16 < qn;                              // a wave without rows only moves tiles
    const auto part_of = [&]() {                                             // [heads, units, buckets], a unit: 16 positions of a sequence
        return k.dpart + (((long)(kvh * k.G + h0 + head)) * k.units + ((long)s * ptiles + ptile) * blocks + blk) * nb;
    };
    if (qn <= 0) {
        if (k.dpart && head < nh) for (int i = lane; i < nb; i += 64) part_of()[i] = 0.f;
        return;
    }
    const T* qb = reinterpret_cast<const T*>(a.q) + (a.q_off ? qr.row0 * a.q_row : s * a.q_seq) + (long)(kvh * k.G + h0) * a.q_head;
    const T* db = reinterpret_cast<const T*>(a.dout) + (a.q_off ? qr.row0 * a.do_row : s * a.do_seq) + (long)(kvh * k.G + h0) * a.do_head;
    const T* ob = reinterpret_cast<const T*>(a.out) + (a.q_off ? qr.row0 * a.o_row : s * a.o_seq) + (long)(kvh * k.G + h0) * a.o_head;
    const T* kb = reinterpret_cast<const T*>(a.k) + (a.k_off ? kr.row0 * a.k_row : s * a.k_seq) + (long)kvh * a.k_head;
    const T* vb = reinterpret_cast<const T*>(a.v) + (a.k_off ? kr.row0 * a.v_row : s * a.v_seq) + (long)kvh * a.v_head;
    const int plo = q0 + shift, phi = q0 + qn - 1 + shift;
    int kend = kr.len;
    if (a.causal && phi + 1 < kend) kend = phi + 1 < 0 ? 0 : phi + 1;

    float vmax = 0.f, own = 0.f;                                             // fp16: max |V_j|^2, |dO_i|^2
    if constexpr (SCALED<T>) {
        for (int i = lane; i < k.n_amax; i += 64) vmax = fmaxf(vmax, k.amax[(long)(s * a.kv_heads + kvh) * k.n_amax + i]);
#pragma unroll
        for (int x = 32; x; x >>= 1) vmax = fmaxf(vmax, __shfl_xor(vmax, x));
    }
    v8<T> qf[Dm::KS], df[Dm::KS];
    const int q = q0 + blk * 16 + li, pos = q + shift;
    const bool row = on && q < qr.len;
    float lse = __builtin_inff(), dl = 0.f, far_lo = 0.f, far_hi = 0.f, sum_lo = 0.f, sum_hi = 0.f;
    const long at_row = (qr.row0 + q) * a.heads + kvh * k.G + h0 + head;
    float dot = 0.f;
#pragma unroll
    for (int ks = 0; ks < Dm::KS; ++ks) {
        qf[ks] = frag_global(qb + q * a.q_row + head * a.q_head, ks * 32 + g4 * 8, D, row);
        df[ks] = frag_global(db + q * a.do_row + head * a.do_head, ks * 32 + g4 * 8, D, row);
        const v8<T> of = frag_global(ob + q * a.o_row + head * a.o_head, ks * 32 + g4 * 8, D, row);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            dot = fmaf((float)df[ks][j], (float)of[j], dot);
            if constexpr (SCALED<T>) own = fmaf((float)df[ks][j], (float)df[ks][j], own);
        }
        if (a.out_lo) {
            if (a.lo_f32) {
                const v8<float> lo = frag_global(reinterpret_cast<const float*>(a.out_lo) + at_row * D, ks * 32 + g4 * 8, D, row);
#pragma unroll
                for (int j = 0; j < 8; ++j) dot = fmaf((float)df[ks][j], lo[j], dot);
            } else {
                const v8<T> lo = frag_global(reinterpret_cast<const T*>(a.out_lo) + at_row * D, ks * 32 + g4 * 8, D, row);
#pragma unroll
                for (int j = 0; j < 8; ++j) dot = fmaf((float)df[ks][j], (float)lo[j], dot);
            }
        }
    }
    dot = sum_over_groups(dot);                                              // D of the row; kept for the other kernel with the exponent to take off
    float up = 1.f, down = 1.f;                                              // factor on the row's dS for the product
    if constexpr (SCALED<T>) {
        const int ex = ds_exponent(sum_over_groups(own) * vmax);
        if (row && g4 == 0) k.row_exp[at_row] = ex;
        up = pow2i(ex); down = pow2i(-ex);
    }
    // A 16-bit product is rounded towards minus infinity more often than up (-2.7e-8 a step of 64 in fp16 beside a result of 8: measured).  In a sum over a
    // bucket such errors add up where dS itself cancels (2e-6 of a gradient at 1500 keys), so every other block of 16 positions works on -dO and D, and its
    // sums change their sign at the end.
    const bool minus = sizeof(T) == 2 && ((q0 >> 4) + blk & 1) != 0;
    if (minus) {
#pragma unroll
        for (int ks = 0; ks < Dm::KS; ++ks) df[ks] = -df[ks];
    }
    if (row) {
        const float e = a.lse[at_row] == NEG_INF ? __builtin_inff() : a.lse[at_row];       // a row that saw no key: every p is 0
        if (g4 == 0) { k.delta[at_row * 2] = e; k.delta[at_row * 2 + 1] = dot; }
        lse = e; dl = minus ? dot : -dot;
    }
    if (k.dpart) {
        for (int i = lane; i < nb; i += 64) bacc[i] = 0.f;
        for (int i = lane; i < WAVE_SUMS; i += 64) order[i] = 0.f;
    }
    if (D < Dm::W) zero_pad_columns<T, Dm::W>(tiles, 4 * BK, PT, D);

    f32x4 o[Dm::ND];
#pragma unroll
    for (int d = 0; d < Dm::ND; ++d) o[d] = (f32x4)(0.f);
    const int krb = (int)a.k_row * (int)sizeof(T), vrb = (int)a.v_row * (int)sizeof(T);
    Stage<T, BK, Dm::W> sk, sv;
    sk.init(krb, D, PT); sv.init(vrb, D, PT);
    int wbeg = 0, wend = 0;
    const int near_lo = plo - a.span - BK + 1, near_hi = a.table ? phi + a.span : near_lo;
    const auto near = [&](int k0) { return k0 > near_lo && k0 < near_hi; };
    const int whole = a.causal && plo + 1 < kr.len ? plo + 1 - BK : kr.len - BK;            // tiles up to here hide no key
    const T *kp = kb, *vp = vb;
    const long kstep = (long)BK * a.k_row, vstep = (long)BK * a.v_row;
    const auto window_for = [&](int k0) {                                    // as in the forward
        if (!near(k0) || k0 + BK + 16 - plo <= wend) return;
        __syncthreads();
        wbeg = k0 - phi - 16; wend = wbeg + k.win;                           // 16 more on either side: lanes without a pair, and sums carried over
        load_window(k, tab, nh, window, wbeg, bwin);
    };
    // sums by offset: lane (g4, x) stands at offset key block - first position + 4 g4 - x
    float acc = 0.f, carry = 0.f;
    int cur = 0, at = 0;                                                     // bucket of acc; key block minus first position when it was last added to
    const auto by_offset = [&](float v) {                                    // sums over the lane groups: of 28 offsets, in lanes 0 .. 27
        order[g4 * 32 + 15 + 4 * g4 - li] = v;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        const int x = lane < 28 ? lane : 28;
        const float sum = (order[x] + order[32 + x]) + (order[64 + x] + order[96 + x]);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        return sum;
    };
    const auto give = [&]() {
        reinterpret_cast<int*>(order)[128 + 15 + 4 * g4 - li] = cur;
        const float v = by_offset(acc);
        const int b = reinterpret_cast<int*>(order)[128 + (lane < 28 ? lane : 28)];
        seq_bucket_runs(v, b, lane < 28, at - 15, bacc);
        acc = 0.f;
    };
    const auto take = [&](float v, int b, int where) {
        const unsigned long long moved = __ballot(b != cur);
        if (moved) {
            const int old = __builtin_amdgcn_readlane(cur, __ffsll(moved) - 1);
            if (__ballot(b != cur && cur != old)) give();
            else {                                                           // one bucket's end, as nearly always far from the diagonal
                const float sum = seq_wave_sum(b != cur ? acc : 0.f);
                if (lane == 0) __hip_atomic_fetch_add(bacc + old, sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);      // an add that nobody waits for
                if (b != cur) acc = 0.f;
            }
            cur = b;
        }
        acc += v; at = where;
    };
    bool open = false, zone = false;                                         // sums are held; sums were added to diag
    const auto close_sums = [&](int k0) {                                    // k0: the key block behind the last one added
        const int where = k0 - (q0 + blk * 16 + shift);
        take(carry, bwin[where + 4 * g4 - li - wbeg], where);
        give();
        carry = 0.f;
        open = false;
    };
    if (kend > 0) {
        const int n = kr.len < BK ? kr.len : BK;
        sk.fetch(kb, n, krb, D); sv.fetch(vb, n, vrb, D);
        if (a.table) {
            load_table(k, kvh * k.G + h0, nh, tab);
            __syncthreads();
            const int blo = seq_bucket(a.map, a.span, nb, -a.span), bhi = seq_bucket(a.map, a.span, nb, a.span);
            if (on) { far_lo = tab[head * nb + blo] * k.c; far_hi = tab[head * nb + bhi] * k.c; }
            wend = -phi;
            window_for(0);
        }
        sk.put(tiles); sv.put(tiles + BK * PT);
    }
#pragma unroll
    for (int ks = 0; ks < Dm::KS; ++ks) { settle(qf[ks]); settle(df[ks]); }
    settle(lse); settle(dl);
    __syncthreads();
    int buf = 0;
    for (int k0 = 0; k0 < kend; k0 += BK) {
        const T* kt = tiles + buf * 2 * BK * PT;
        const T* vt = kt + BK * PT;
        const int next = k0 + BK;
        if (next < kend) {
            const int n = kr.len - next < BK ? kr.len - next : BK;
            kp += kstep; vp += vstep;
            sk.fetch(kp, n, krb, D);
            sv.fetch(vp, n, vrb, D);
        }
        if (on) {
            const bool close = near(k0), high = k0 >= phi;
            f32x4 sc[NB], dp[NB];
            float sub = -lse;
            v8<T> kf[NB][Dm::KS], vf[NB][Dm::KS];
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int ks = 0; ks < Dm::KS; ++ks) kf[n][ks] = frag_row(kt + (n * 16 + li) * PT + ks * 32 + g4 * 8);
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int ks = 0; ks < Dm::KS; ++ks) vf[n][ks] = frag_row(vt + (n * 16 + li) * PT + ks * 32 + g4 * 8);
            if (close) {
                const int p = pos <= phi ? pos : phi;
                const float* sp = reinterpret_cast<const float*>(lds) + whole_index((int)(window - reinterpret_cast<float*>(lds)) + head * k.win + (k0 - wbeg - p) + 4 * g4);
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) sc[n][r] = sp[n * 16 + r];
            } else {
                sub += high ? far_hi : far_lo;
#pragma unroll
                for (int n = 0; n < NB; ++n) sc[n] = (f32x4)(0.f);
            }
#pragma unroll
            for (int n = 0; n < NB; ++n) dp[n] = (f32x4)(dl);
            ahead<T>();
#pragma unroll
            for (int ks = 0; ks < Dm::KS; ++ks)
#pragma unroll
                for (int n = 0; n < NB; ++n) sc[n] = Seq<T>::mma(kf[n][ks], qf[ks], sc[n]);
#pragma unroll
            for (int ks = 0; ks < Dm::KS; ++ks)
#pragma unroll
                for (int n = 0; n < NB; ++n) dp[n] = Seq<T>::mma(vf[n][ks], df[ks], dp[n]);
            v8<T> kc[NB / 2][Dm::ND];                                        // on their way behind the exponentials
#pragma unroll
            for (int u = 0; u < NB / 2; ++u)
#pragma unroll
                for (int d = 0; d < Dm::ND; ++d) kc[u][d] = frag_col(kt, PT, u * 32, d * 16, g4, li);
            ahead<T>();
            if (k0 > whole) {
                const int lim = (a.causal && pos < kr.len - 1 ? pos : kr.len - 1) - k0 - 4 * g4;
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (n * 16 + r > lim) sc[n][r] = NEG_INF;
            }
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) sc[n][r] = exp2_hw(fmaf(sc[n][r], k.c, sub)) * dp[n][r];
            if (k.dpart && !close) {
                float sum = 0.f;
#pragma unroll
                for (int n = 0; n < NB; ++n) sum += (sc[n][0] + sc[n][1]) + (sc[n][2] + sc[n][3]);
                if (high) sum_hi += sum; else sum_lo += sum;
                if (open) close_sums(k0);
            } else if (k.dpart) {
                open = true;
                const int where = k0 - (q0 + blk * 16 + shift);
                float v[NB];
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    const f32x4 x = sc[n];
                    v[n] = carry + x[0] + dpp_shift<0x101>(x[1]) + (dpp_shift<0x102>(x[2]) + dpp_shift<0x103>(x[3]));
                    carry = dpp_shift<0x11d>(x[3] + (dpp_shift<0x111>(x[2]) + dpp_shift<0x112>(x[1])));
                }
                if (where >= -ZONE && where + (NB - 1) * 16 <= ZONE) {
#pragma unroll
                    for (int n = 0; n < NB; ++n) {
                        const float sum = by_offset(v[n]);
                        if (lane < 28) diag[ZONE + where + n * 16 + lane] += sum;
                    }
                    zone = true;
                } else {
                    const uint8_t* bw = bwin + (where + 4 * g4 - li - wbeg);
                    int b[NB];
                    bool same = true;
#pragma unroll
                    for (int n = 0; n < NB; ++n) { b[n] = bw[n * 16]; same = same && b[n] == cur; }
                    if (__all(same)) {
#pragma unroll
                        for (int n = 0; n < NB; ++n) acc += v[n];
                        at = where + (NB - 1) * 16;
                    } else {
#pragma unroll
                        for (int n = 0; n < NB; ++n) take(v[n], b[n], where + n * 16);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < NB / 2; ++u) {
                if constexpr (SCALED<T>) { sc[2 * u] *= up; sc[2 * u + 1] *= up; }
                const v8<T> pf = frag_acc<T>(sc[2 * u], sc[2 * u + 1]);      // dS rounded to T once, for the product only
#pragma unroll
                for (int d = 0; d < Dm::ND; ++d) o[d] = mma_sum<T>(kc[u][d], pf, o[d]);
            }
        }
        if (next < kend) {
            buf ^= 1;
            sk.put(tiles + buf * 2 * BK * PT); sv.put(tiles + (buf * 2 + 1) * BK * PT);
            window_for(next);
        }
        __syncthreads();
    }
    const float sign = minus ? -1.f : 1.f;
    if (k.dpart) {
        if (on && open) close_sums((kend + BK - 1) / BK * BK);
        if (zone)
            for (int c = 0; c < 2 * ZONE + 32; c += 64) {
                const int first = c - ZONE - 15;
                seq_bucket_runs(diag[c + lane], seq_bucket(a.map, a.span, nb, first + lane), true, first, bacc);
            }
        const int blo = seq_bucket(a.map, a.span, nb, -a.span), bhi = seq_bucket(a.map, a.span, nb, a.span);
        const float lo = seq_wave_sum(sum_lo), hi = seq_wave_sum(sum_hi);
        if (lane == 0) { bacc[blo] += lo; bacc[bhi] += hi; }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (head < nh) for (int i = lane; i < nb; i += 64) part_of()[i] = bacc[i] * sign;
    }
    if (!row) return;
    T* dst = reinterpret_cast<T*>(a.dq) + at_row * D;
    typedef T t4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int d = 0; d < Dm::ND; ++d) {
        const int c = d * 16 + g4 * 4;
        if (c >= D) continue;
        t4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = (T)(o[d][j] * (a.scale * (sign * down)));
        *reinterpret_cast<t4*>(dst + c) = v;
    }
}

// dK and dV.  4 waves, wave w owns keys [16 MK w, 16 MK (w + 1)) of the tile and walks the query rows BQ at a time; S and dP [query][key] with the K and V
// fragments in registers, dV^T += dO^T P, dK^T += Q^T dS.
// PAIR: wide heads of 16-bit types have no registers for more than 16 keys a wave, and then four fragments come out of LDS for four products.  So two
// waves share 32 keys: one holds K and dV, the other V and dK, and every fragment serves two products.  P goes from one to the other through
// LDS in fp32, a tile behind, and the products of dV run a tile behind, too, under the exponentials of the next.  (Dense 4 x 16 heads x 2048 x
// 128, whole backward: 710 us, 743 with 16 keys a wave; causal 32 heads x 8192: 2330, 2530.)
// The rows are walked from the last to the first, so that the causal tiles of keys read the same rows at a time.
template <typename T, int DT, int MK, int BQ, bool PAIR>
__global__ __launch_bounds__(256, grad_waves<T>(DT)) void rel_attn_dkv_kernel(const RelAttn k) {
    typedef Dims<DT> Dm;
    typedef int i32x4 __attribute__((ext_vector_type(4)));
    constexpr int BKV = PAIR ? 64 : 64 * MK, NQ = BQ / 16, PT = pitch_of<T>(Dm::W), QB = PAIR ? 3 : 2, PW = NQ * MK * 256;
    extern __shared__ __attribute__((aligned(32))) char lds[];
    const cv_rel_attn& a = k.a;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g4 = lane >> 4, li = lane & 15;
    T* tiles = reinterpret_cast<T*>(lds);                                    // QB of Q, 2 of dO
    float* rowv = reinterpret_cast<float*>(tiles + (QB + 2) * BQ * PT);      // of a tile's rows: exponent to add, -D, window index, position; twice
    int* tile_exp = reinterpret_cast<int*>(rowv + 8 * BQ);                   // fp16: exponents of the two tiles of rows
    float* pass = rowv + 8 * BQ + 4;                                         // pairs: P on its way to the other wave, [2][2 pairs]
    float* tab = pass + (PAIR ? 4 * PW : 0);
    float* window = tab + k.G * a.num_buckets;

    Part me;
    if (!part_of_block(k, me)) return;
    const int tile = me.tile, kvh = me.kvh, s = me.s;
    if (a.k_off && a.zero_rest && tile + kvh == 0) {
        const long row = (long)a.kv_heads * a.head_dim;
        zero_rest(a.k_off, s, a.n_seq, a.max_k, a.rows_k, reinterpret_cast<T*>(a.dk), row, a.kv_heads, a.head_dim, a.head_dim);
        zero_rest(a.k_off, s, a.n_seq, a.max_k, a.rows_k, reinterpret_cast<T*>(a.dv), row, a.kv_heads, a.head_dim, a.head_dim);
    }
    const SeqRange qr = seq_range(a.q_off, s, a.max_q, a.rows_q), kr = seq_range(a.k_off, s, a.max_k, a.rows_k);
    const int c0 = tile * BKV, shift = kr.len - qr.len, D = a.head_dim;
    if (c0 >= kr.len) return;
    const T* qb = reinterpret_cast<const T*>(a.q) + (a.q_off ? qr.row0 * a.q_row : s * a.q_seq) + (long)kvh * k.G * a.q_head;
    const T* db = reinterpret_cast<const T*>(a.dout) + (a.q_off ? qr.row0 * a.do_row : s * a.do_seq) + (long)kvh * k.G * a.do_head;
    const T* kb = reinterpret_cast<const T*>(a.k) + (a.k_off ? kr.row0 * a.k_row : s * a.k_seq) + (long)kvh * a.k_head;
    const T* vb = reinterpret_cast<const T*>(a.v) + (a.k_off ? kr.row0 * a.v_row : s * a.v_seq) + (long)kvh * a.v_head;
    const int clast = (c0 + BKV < kr.len ? c0 + BKV : kr.len) - 1;
    int qbeg = 0;                                                            // causal: rows before the first that sees key c0 are skipped
    if (a.causal && c0 > shift) { qbeg = c0 - shift < qr.len ? c0 - shift : qr.len; qbeg -= qbeg % k.qt; }
    const int qfirst = (qr.len + k.qt - 1) / k.qt * k.qt - k.qt;             // from the last rows to the first: the tiles of keys read the same rows at a time
    int ex = DS_FREE;                                                        // fp16: dK holds 2^ex of its value
    float up = pow2i(ex - P_UP<T>);                                          // from P 2^P_UP (dP - D)
    const int role = PAIR ? __builtin_amdgcn_readfirstlane((wave >> 1) ^ (int)(blockIdx.x >> 8 & 1)) : 0, part = PAIR ? wave & 1 : wave;
    v8<T> kf[MK][Dm::KS], vf[PAIR ? 1 : MK][Dm::KS];                         // pairs: kf holds K or V
    int key[MK];
#pragma unroll
    for (int m = 0; m < MK; ++m) {
        key[m] = c0 + (part * MK + m) * 16 + li;
#pragma unroll
        for (int ks = 0; ks < Dm::KS; ++ks) {
            kf[m][ks] = frag_global(role ? vb + key[m] * a.v_row : kb + key[m] * a.k_row, ks * 32 + g4 * 8, D, key[m] < kr.len);
            if constexpr (!PAIR) vf[m][ks] = frag_global(vb + key[m] * a.v_row, ks * 32 + g4 * 8, D, key[m] < kr.len);
        }
    }
    const bool busy = c0 + part * MK * 16 < kr.len;
    if (D < Dm::W) zero_pad_columns<T, Dm::W>(tiles, (QB + 2) * BQ, PT, D);
    f32x4 dk[MK][Dm::ND], dv[PAIR ? 1 : MK][Dm::ND];                         // pairs: dk holds dK or dV
#pragma unroll
    for (int m = 0; m < MK; ++m)
#pragma unroll
        for (int d = 0; d < Dm::ND; ++d) {
            dk[m][d] = (f32x4)(0.f);
            if constexpr (!PAIR) dv[m][d] = (f32x4)(0.f);
        }

    Stage<T, BQ, Dm::W> sq, sd;
    sq.init_rows((int)a.q_row * (int)sizeof(T), (int)a.q_head * (int)sizeof(T), k.G, k.rt, D, PT);
    sd.init_rows((int)a.do_row * (int)sizeof(T), (int)a.do_head * (int)sizeof(T), k.G, k.rt, D, PT);
    float2 st = {__builtin_inff(), 0.f};
    int se = DS_FREE;
    const float2* stats = reinterpret_cast<const float2*>(k.delta) + qr.row0 * a.heads + kvh * k.G;
    const int my_qi = (int)threadIdx.x / k.G, my_g = (int)threadIdx.x - my_qi * k.G;       // of the tile's row threadIdx.x
    const long qstep = k.qt * a.q_row, dstep = k.qt * a.do_row, sstep = (long)k.qt * a.heads;
    const T *qp = qb + qfirst * a.q_row, *dp_ = db + qfirst * a.do_row;
    const float2* sp = stats + (long)(qfirst + my_qi) * a.heads + my_g;
    const int* ep = k.row_exp + (sp - reinterpret_cast<const float2*>(k.delta));
    const auto fetch = [&](int q0) {                                         // the tiles come one after the other
        const int n = qr.len - q0 < k.qt ? (qr.len - q0) * k.G : k.rt;
        sq.fetch_rows(qp, n, PT);
        sd.fetch_rows(dp_, n, PT);
        if (threadIdx.x < BQ) st = (int)threadIdx.x < n ? *sp : float2{__builtin_inff(), 0.f};
        if constexpr (SCALED<T>) {
            if (threadIdx.x < BQ) se = (int)threadIdx.x < n ? *ep : DS_FREE;
            ep -= sstep;
        }
        qp -= qstep; dp_ -= dstep; sp -= sstep;
    };
    // offsets a tile of rows meets: c0 - phi .. c0 + BKV - 1 - plo
    int wbeg = 0, wend = 0x80000000;
    float far_lo = 0.f, far_hi = 0.f;
    const auto last_of = [&](int q0) { return (q0 + k.qt < qr.len ? q0 + k.qt : qr.len) - 1; };
    const auto near = [&](int q0) { return a.table && c0 - shift - last_of(q0) < a.span && clast - shift - q0 > -a.span; };
    const auto put = [&](int q0, int buf, int qbuf) {                                  // every wave is past the products that read this buffer and the window
        const int plo = q0 + shift, phi = last_of(q0) + shift;
        const bool close = near(q0);
        sq.put(tiles + qbuf * BQ * PT); sd.put(tiles + (QB + buf) * BQ * PT);
        if (close && c0 + BKV - plo > wend) {
            __syncthreads();
            wbeg = c0 - phi; wend = wbeg + k.win;
            load_window(k, tab, k.G, window, wbeg);
        }
        if (threadIdx.x < BQ) {
            const int pos = plo + my_qi;
            float* v = rowv + buf * 4 * BQ + threadIdx.x;
            v[0] = (close || !a.table ? 0.f : c0 >= phi ? far_hi : far_lo) - (st.x - (float)P_UP<T>);
            v[BQ] = -st.y;
            reinterpret_cast<int*>(v)[2 * BQ] = close && pos <= phi ? my_g * k.win - pos - wbeg : -c0;   // + key; rows past the end read word 0 on
            reinterpret_cast<int*>(v)[3 * BQ] = pos;
            if constexpr (SCALED<T>) {                                       // the smallest over the tile's 32 rows, in lane 31
                static_assert(BQ == 32, "a half wave holds a tile's rows");
                int e = se;
                e = dpp_min<0x111, 0xf>(e); e = dpp_min<0x112, 0xf>(e); e = dpp_min<0x114, 0xf>(e); e = dpp_min<0x118, 0xf>(e);
                e = dpp_min<0x142, 0x2>(e);
                if (threadIdx.x == 31) tile_exp[buf] = e;
            }
        }
    };
    // fp16: before a tile's dS is added.  Where its rows need a smaller factor, what was added before takes it, too (a power of two: exact).
    const auto follow = [&](int e) {
        if (e >= ex) return;
        const float f = pow2i(e - ex);
        ex = e; up = pow2i(e - P_UP<T>);
#pragma unroll
        for (int m = 0; m < MK; ++m)
#pragma unroll
            for (int d = 0; d < Dm::ND; ++d) dk[m][d] *= f;
    };
    const auto exponent_of = [&](int buf) { return SCALED<T> ? __builtin_amdgcn_readfirstlane(tile_exp[buf]) : 0; };
    if (qbeg < qr.len) {
        fetch(qfirst);
        if (a.table) {
            load_table(k, kvh * k.G, k.G, tab);
            __syncthreads();
            const int g = my_g < k.G ? my_g : 0;
            far_lo = tab[g * a.num_buckets + seq_bucket(a.map, a.span, a.num_buckets, -a.span)] * k.c;
            far_hi = tab[g * a.num_buckets + seq_bucket(a.map, a.span, a.num_buckets, a.span)] * k.c;
        }
        put(qfirst, 0, 0);
    }
#pragma unroll
    for (int m = 0; m < MK; ++m)
#pragma unroll
        for (int ks = 0; ks < Dm::KS; ++ks) {
            settle(kf[m][ks]);
            if constexpr (!PAIR) settle(vf[m][ks]);
        }
    __syncthreads();
    const auto read_rows = [&](const T* tile, v8<T> (&f)[NQ][Dm::KS]) {
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int ks = 0; ks < Dm::KS; ++ks) f[n][ks] = frag_row(tile + (n * 16 + li) * PT + ks * 32 + g4 * 8);
    };
    const auto read_cols = [&](const T* tile, v8<T> (&f)[NQ / 2][Dm::ND]) {
#pragma unroll
        for (int u = 0; u < NQ / 2; ++u)
#pragma unroll
            for (int d = 0; d < Dm::ND; ++d) f[u][d] = frag_col(tile, PT, u * 32, d * 16, g4, li);
    };
    const auto biases = [&](const float* rv, int q0, f32x4 (&sc)[NQ][MK]) {             // what the products of S start from
        const bool close = near(q0);
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
#pragma unroll
            for (int m = 0; m < MK; ++m) sc[n][m] = (f32x4)(0.f);
            if (close) {
                const i32x4 at = *reinterpret_cast<const i32x4*>(rv + 2 * BQ + n * 16);
#pragma unroll
                for (int m = 0; m < MK; ++m)
#pragma unroll
                    for (int r = 0; r < 4; ++r) sc[n][m][r] = window[at[r] + key[m]];
            }
        }
    };
    const auto minus_d = [&](const float* rv, f32x4 (&dp)[NQ][MK]) {                    // what the products of dP start from
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int m = 0; m < MK; ++m) dp[n][m] = *reinterpret_cast<const f32x4*>(rv + BQ + n * 16);
    };
    const auto products = [&](const v8<T> (&rows)[NQ][Dm::KS], const auto& keys, f32x4 (&acc)[NQ][MK]) {
#pragma unroll
        for (int ks = 0; ks < Dm::KS; ++ks)
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
                for (int m = 0; m < MK; ++m) acc[n][m] = Seq<T>::mma(rows[n][ks], keys[m][ks], acc[n][m]);
    };
    const auto weights = [&](const float* rv, int q0, f32x4 (&sc)[NQ][MK]) {            // S -> P 2^P_UP
        if (a.causal && clast > q0 + shift) {
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                const i32x4 ps = *reinterpret_cast<const i32x4*>(rv + 3 * BQ + n * 16);
#pragma unroll
                for (int m = 0; m < MK; ++m)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (key[m] > ps[r]) sc[n][m][r] = NEG_INF;
            }
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const f32x4 sub = *reinterpret_cast<const f32x4*>(rv + n * 16);
#pragma unroll
            for (int m = 0; m < MK; ++m)
#pragma unroll
                for (int r = 0; r < 4; ++r) sc[n][m][r] = exp2_hw(fmaf(sc[n][m][r], k.c, sub[r]));
        }
    };
    const auto scaled = [&](const f32x4 (&p)[NQ][MK], f32x4 (&dp)[NQ][MK]) {            // dP - D -> dS
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int m = 0; m < MK; ++m)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float d = p[n][m][r] * dp[n][m][r];
                    if constexpr (SCALED<T>) d *= up;
                    dp[n][m][r] = d;
                }
    };
    const auto rounded = [&](const f32x4 (&x)[NQ][MK], v8<T> (&f)[NQ / 2][MK]) {        // P and dS rounded to T once, for the products only
#pragma unroll
        for (int u = 0; u < NQ / 2; ++u)
#pragma unroll
            for (int m = 0; m < MK; ++m) f[u][m] = frag_acc<T>(x[2 * u][m], x[2 * u + 1][m]);
    };
    // body(Q tile, dO tile, row values, buffer, first row); the next tile's loads run behind it
    const auto walk = [&](auto body) {
        int buf = 0, qbuf = 0;
        for (int q0 = qfirst; q0 >= qbeg; q0 -= k.qt) {
            const int next = q0 - k.qt;
            if (next >= qbeg) fetch(next);
            if (busy) body(tiles + qbuf * BQ * PT, tiles + (QB + buf) * BQ * PT, rowv + buf * 4 * BQ + g4 * 4, buf, q0);
            buf ^= 1; qbuf = qbuf == QB - 1 ? 0 : qbuf + 1;
            if (next >= qbeg) put(next, buf, qbuf);
            __syncthreads();
        }
    };
    if constexpr (!PAIR) {
        walk([&](const T* qt, const T* dt, const float* rv, int buf, int q0) {
            if constexpr (SCALED<T>) follow(exponent_of(buf));
            f32x4 sc[NQ][MK], dp[NQ][MK];
            v8<T> qf[NQ][Dm::KS], df[NQ][Dm::KS];
            read_rows(qt, qf);
            read_rows(dt, df);
            biases(rv, q0, sc);
            minus_d(rv, dp);
            ahead<T>();
            products(qf, kf, sc);
            products(df, vf, dp);
            v8<T> qc[NQ / 2][Dm::ND], dc[NQ / 2][Dm::ND], pf[NQ / 2][MK], sf[NQ / 2][MK];
            read_cols(dt, dc);                                               // on their way behind the exponentials
            read_cols(qt, qc);
            ahead<T>();
            weights(rv, q0, sc);
            scaled(sc, dp);
            rounded(sc, pf);
            rounded(dp, sf);
#pragma unroll
            for (int u = 0; u < NQ / 2; ++u)
#pragma unroll
                for (int d = 0; d < Dm::ND; ++d)
#pragma unroll
                    for (int m = 0; m < MK; ++m) {
                        dv[m][d] = mma_sum<T>(dc[u][d], pf[u][m], dv[m][d]);
                        dk[m][d] = mma_sum<T>(qc[u][d], sf[u][m], dk[m][d]);
                    }
        });
    } else if (role == 0) {
        v8<T> dc[NQ / 2][Dm::ND], pf[NQ / 2][MK];                            // of the tile before: its products run behind this one's exponentials
#pragma unroll
        for (int u = 0; u < NQ / 2; ++u) {
#pragma unroll
            for (int d = 0; d < Dm::ND; ++d) dc[u][d] = frag_zero<T>();
#pragma unroll
            for (int m = 0; m < MK; ++m) pf[u][m] = frag_zero<T>();
        }
        const auto value_gradient = [&]() {
#pragma unroll
            for (int u = 0; u < NQ / 2; ++u)
#pragma unroll
                for (int d = 0; d < Dm::ND; ++d)
#pragma unroll
                    for (int m = 0; m < MK; ++m) dk[m][d] = Seq<T>::mma(dc[u][d], pf[u][m], dk[m][d]);
        };
        walk([&](const T* qt, const T* dt, const float* rv, int buf, int q0) {
            f32x4 sc[NQ][MK];
            v8<T> qf[NQ][Dm::KS];
            read_rows(qt, qf);
            biases(rv, q0, sc);
            ahead<T>();
            products(qf, kf, sc);
            value_gradient();
            weights(rv, q0, sc);
#pragma unroll
            for (int i = 0; i < 2 * Dm::ND; ++i) { __builtin_amdgcn_sched_group_barrier(8, 1, 0); __builtin_amdgcn_sched_group_barrier(2, 4, 0); }    // a product, four VALU instructions, ...
            read_cols(dt, dc);
            float* to = pass + (buf * 2 + part) * PW;
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
                for (int m = 0; m < MK; ++m) *reinterpret_cast<f32x4*>(to + ((n * MK + m) * 64 + lane) * 4) = sc[n][m];
            rounded(sc, pf);
        });
        value_gradient();
    } else {
        f32x4 dp[NQ][MK];
        const T* qlast = tiles;
        int last = -1, last_exp = DS_FREE;
        const auto key_gradient = [&]() {                                    // dK of the tile before, with the P that the other wave left
            if constexpr (SCALED<T>) follow(last_exp);
            f32x4 p[NQ][MK];
            const float* from = pass + (last * 2 + part) * PW;
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
                for (int m = 0; m < MK; ++m) p[n][m] = *reinterpret_cast<const f32x4*>(from + ((n * MK + m) * 64 + lane) * 4);
            v8<T> qc[NQ / 2][Dm::ND], sf[NQ / 2][MK];
            read_cols(qlast, qc);
            scaled(p, dp);
            rounded(dp, sf);
#pragma unroll
            for (int u = 0; u < NQ / 2; ++u)
#pragma unroll
                for (int d = 0; d < Dm::ND; ++d)
#pragma unroll
                    for (int m = 0; m < MK; ++m) dk[m][d] = Seq<T>::mma(qc[u][d], sf[u][m], dk[m][d]);
        };
        walk([&](const T* qt, const T* dt, const float* rv, int buf, int) {
            v8<T> df[NQ][Dm::KS];
            f32x4 now[NQ][MK];
            read_rows(dt, df);
            minus_d(rv, now);
            if (last >= 0) key_gradient();
            products(df, kf, now);
#pragma unroll
            for (int n = 0; n < NQ; ++n)
#pragma unroll
                for (int m = 0; m < MK; ++m) dp[n][m] = now[n][m];
            qlast = qt; last = buf;
            last_exp = exponent_of(buf);
        });
        if (last >= 0) key_gradient();
    }
#pragma unroll
    for (int m = 0; m < MK; ++m) {
        if (key[m] >= kr.len) continue;
        const float back = SCALED<T> ? pow2i(-ex) : 1.f;
        const long at = ((kr.row0 + key[m]) * a.kv_heads + kvh) * D;
        typedef T t4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int d = 0; d < Dm::ND; ++d) {
            const int c = d * 16 + g4 * 4;
            if (c >= D) continue;
            t4 x, y;
            if constexpr (PAIR) {
                const float f = role ? a.scale * back : pow2i(-P_UP<T>);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = (T)(dk[m][d][j] * f);
                *reinterpret_cast<t4*>(reinterpret_cast<T*>(role ? a.dk : a.dv) + at + c) = x;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) { x[j] = (T)(dk[m][d][j] * (a.scale * back)); y[j] = (T)(SCALED<T> ? dv[m][d][j] * pow2i(-P_UP<T>) : dv[m][d][j]); }
                *reinterpret_cast<t4*>(reinterpret_cast<T*>(a.dk) + at + c) = x;
                *reinterpret_cast<t4*>(reinterpret_cast<T*>(a.dv) + at + c) = y;
            }
        }
    }
}

// dtable[b, h] = sum over units of dpart[h, unit, b]: 1024 threads as `wide` buckets x 1024 / wide unit lanes, joined in LDS in a fixed order
__global__ __launch_bounds__(1024) void rel_dtable_kernel(const RelAttn k, int wide) {
    __shared__ float red[1024];
    const cv_rel_attn& a = k.a;
    const int nb = a.num_buckets, h = blockIdx.x, x = threadIdx.x & (wide - 1), lanes = 1024 / wide;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (x < nb) {
        const float* src = k.dpart + (long)h * k.units * nb + x;
        int u = (int)threadIdx.x / wide;
        for (; u + 7 * lanes < k.units; u += 8 * lanes) {
#pragma unroll
            for (int q = 0; q < 8; ++q) acc[q] += src[(long)(u + q * lanes) * nb];
        }
        for (; u < k.units; u += lanes) acc[0] += src[(long)u * nb];
    }
    red[threadIdx.x] = ((acc[0] + acc[1]) + (acc[2] + acc[3])) + ((acc[4] + acc[5]) + (acc[6] + acc[7]));
    for (int n = 512; n >= wide; n >>= 1) {
        __syncthreads();
        if (threadIdx.x < n) red[threadIdx.x] += red[threadIdx.x + n];
    }
    if (threadIdx.x < nb) table_set(a.dtable, a.table_dtype, (long)threadIdx.x * a.heads + h, red[threadIdx.x]);
}

// dQ: one block of 16 rows a wave; two would halve the LDS reads a product, but take 212 .. 256 registers and leave two waves a SIMD instead of four (ragged
// training step, 24 x 12 heads of 64: 660 us with two blocks, 612 with one; causal, heads of 128: 1305, with spills, and 1079).
constexpr int BK_DQ = 32, BQ_DKV = 32;

struct BwdPlan { int keys, ht, q_rt, q_tiles, k_tiles, n_amax; long rows, units; int64_t stat, exps, amax, part; };
BwdPlan bwd_plan(const cv_rel_attn& a) {
    BwdPlan p;
    const int G = a.heads / a.kv_heads;
    p.keys = a.dtype != CV_DTYPE_F32 && a.head_dim <= 64 ? 128 : 64;          // of a dK / dV tile
    p.ht = G < 4 ? G : 4;                                                    // heads of a dQ tile of 4 blocks of 16 rows, and its positions
    p.q_rt = 4 / p.ht * 16;
    const int q_parts = (a.max_q + p.q_rt - 1) / p.q_rt;
    p.q_tiles = q_parts * ((G + p.ht - 1) / p.ht);
    p.k_tiles = (a.max_k + p.keys - 1) / p.keys;
    p.rows = a.q_off ? a.rows_q : (long)a.n_seq * a.max_q;
    const bool scaled = a.dtype == CV_DTYPE_F16;
    const int64_t pairs = (int64_t)a.n_seq * a.kv_heads;                     // parts of a pair: until there are about 1024 workgroups of 64 rows or more
    const long share = pairs < 1 ? 1 : pairs < 1024 ? 1024 / pairs : 1, runs = (a.max_k + 63L) / 64;
    p.n_amax = (int)(runs < share ? (runs < 1 ? 1 : runs) : share);
    p.units = (long)a.n_seq * q_parts * (p.q_rt / 16);
    const auto round = [](int64_t n) { return (n + 15) / 16 * 16; };
    p.stat = round(p.rows * a.heads * 8);
    p.exps = scaled ? round(p.rows * a.heads * 4) : 0;
    p.amax = scaled ? round(pairs * p.n_amax * 4) : 0;
    p.part = a.dtable ? round(p.units * a.heads * (int64_t)a.num_buckets * 4) : 0;
    return p;
}

template <typename T, int DT>
int bwd_launch(RelAttn& k, const BwdPlan& p, hipStream_t st) {
    constexpr bool PAIR = sizeof(T) == 2 && DT > 64;
    constexpr int MK = sizeof(T) == 2 ? 2 : 1;
    const cv_rel_attn& a = k.a;
    const int G = k.G;
    int rc = 0;
    if constexpr (SCALED<T>) {
        if (p.q_tiles > 0 && a.n_seq > 0) {
            hipLaunchKernelGGL((rel_vnorm_kernel<T>), dim3((unsigned)(a.n_seq * a.kv_heads * p.n_amax)), dim3(256), 0, st, k);
            if ((rc = (int)hipGetLastError())) return rc;
        }
    }
    const size_t tabs = a.table ? (size_t)G * a.num_buckets : 0;
    if (p.q_tiles > 0 && a.n_seq > 0) {
        k.tiles = p.q_tiles; k.qt = p.q_rt; k.ht = p.ht;
        k.win = a.table ? window_size(a, p.ht, BK_DQ + p.q_rt + 32) : 0;
        const size_t floats = (size_t)p.ht * (k.a.num_buckets + k.win) + k.win / 4 + (k.dpart ? (size_t)4 * (k.a.num_buckets + WAVE_SUMS) : 0);
        const size_t bytes = 4 * BK_DQ * pitch_of<T>(Dims<DT>::W) * sizeof(T) + floats * 4;
        if ((rc = allow_lds(&rel_attn_dq_kernel<T, DT, BK_DQ>, bytes))) return rc;
        hipLaunchKernelGGL((rel_attn_dq_kernel<T, DT, BK_DQ>), dim3(part_grid(k)), dim3(256), bytes, st, k);
        if ((rc = (int)hipGetLastError())) return rc;
    }
    if (p.k_tiles > 0 && a.n_seq > 0) {
        k.tiles = p.k_tiles; k.rt = BQ_DKV / G * G; k.qt = BQ_DKV / G;
        const auto kernel = &rel_attn_dkv_kernel<T, DT, MK, BQ_DKV, PAIR>;
        k.win = a.table ? window_size(a, G, p.keys + BQ_DKV / G) : 0;
        const size_t bytes = (PAIR ? 5 : 4) * BQ_DKV * pitch_of<T>(Dims<DT>::W) * sizeof(T) + (8 * BQ_DKV + 4 + (PAIR ? 4 * BQ_DKV * 32 : 0) + tabs + (size_t)G * k.win) * 4;
        if ((rc = allow_lds(kernel, bytes))) return rc;
        hipLaunchKernelGGL(kernel, dim3(part_grid(k)), dim3(256), bytes, st, k);
        if ((rc = (int)hipGetLastError())) return rc;
    }
    if (k.dpart) {
        int wide = 8;
        while (wide < a.num_buckets) wide *= 2;
        hipLaunchKernelGGL(rel_dtable_kernel, dim3(a.heads), dim3(1024), 0, st, k, wide);
        rc = (int)hipGetLastError();
    }
    return rc;
}
template <typename T> int bwd_t(RelAttn& k, const BwdPlan& p, hipStream_t st) {
    const int D = k.a.head_dim;
    if (D <= 32) return bwd_launch<T, 32>(k, p, st);
    if (D <= 64) return bwd_launch<T, 64>(k, p, st);
    if (D <= 80) return bwd_launch<T, 80>(k, p, st);
    if (D <= 96) return bwd_launch<T, 96>(k, p, st);
    return bwd_launch<T, 128>(k, p, st);
}

}  // namespace

int64_t rel_attention_bwd_tiles(const cv_rel_attn& a) {
    const BwdPlan p = bwd_plan(a);
    return p.q_tiles > p.k_tiles ? p.q_tiles : p.k_tiles;
}
int64_t rel_attention_bwd_ws(const cv_rel_attn& a) {
    const BwdPlan p = bwd_plan(a);
    return p.stat + p.exps + p.amax + p.part + 16;                           // (never 0)
}

int launch_rel_attention_grad(const cv_rel_attn& a, hipStream_t st) {
    const BwdPlan p = bwd_plan(a);
    const long D = a.head_dim;
    int rc = 0;
    if (a.zero_rest && a.q_off && (a.n_seq == 0 || a.max_q == 0) && (rc = launch_rel_zero(a.dq, a.dtype, a.rows_q, a.heads, a.head_dim, a.heads * D, D, st))) return rc;
    if (a.zero_rest && a.k_off && (a.n_seq == 0 || a.max_k == 0))
        for (void* t : {a.dk, a.dv})
            if ((rc = launch_rel_zero(t, a.dtype, a.rows_k, a.kv_heads, a.head_dim, a.kv_heads * D, D, st))) return rc;
    RelAttn k{};
    k.a = a; k.G = a.heads / a.kv_heads; k.nsplit = 1; k.c = a.scale * LOG2E;
    if (!a.table) k.a.num_buckets = 0;
    char* ws = reinterpret_cast<char*>(a.ws);
    k.delta = reinterpret_cast<float*>(ws);
    k.row_exp = reinterpret_cast<int*>(ws + p.stat);
    k.amax = reinterpret_cast<float*>(ws + p.stat + p.exps); k.n_amax = p.n_amax;
    k.dpart = a.dtable ? reinterpret_cast<float*>(ws + p.stat + p.exps + p.amax) : nullptr;
    k.units = (int)p.units;
    return a.dtype == CV_DTYPE_F16 ? bwd_t<half_t>(k, p, st) : a.dtype == CV_DTYPE_BF16 ? bwd_t<bhalf_t>(k, p, st) : bwd_t<float>(k, p, st);
}

}  // namespace cva
