// Attention with a bucketed position bias, forward:  o_i = sum_j softmax_j(scale q_i . k_j + t[map(j - pos_i), head]) v_j.
// One pass over the keys with a running maximum and sum; the bias enters as the starting value of the S^T accumulators, read from a window of
// offsets in LDS; in a tile beyond the span on either side it is one exponent a row.
// Bound by the matrix pipe and the exponentials for long rows, by HBM (K and V once) for single tokens.
// Few rows: the keys are split over workgroups and a second kernel joins the parts.
#include "relattn.h"

namespace cva {
namespace {

// 4 waves, wave w owns rows [16 MQ w, 16 MQ (w + 1)) of the tile; BK keys a step, two LDS buffers: the loads of the next tile run behind the products of
// this one, one barrier a tile.  Heads up to 64 wide: three waves a SIMD hide more than fragments read ahead (ragged training step: 561 us, 585 with
// two waves and all fragments ahead); wider ones have registers for two waves at most.
// 8 x 16 heads x 4096 x 80 fp16: 880 to 900 us, 770 TFLOP/s; bound by issue: a 16 x 16 block takes a SIMD 232 cycles, 88 of products (heads padded to 96 in
// the first) and 129 of VALU, half of that the exponentials; the two waves of a SIMD overlap them little.
// REST (training): the sums of what rounding P left, too.  The parts cost VALU (three to four instructions an element in fp16, five in bf16) and products: 24 x 12 heads
// x up to 1500 x 64 bf16 198 us, 114 without; causal 2 x 16 x 4096 x 128 fp16 260, 203.  The second set of accumulators leaves two waves a SIMD for heads up to
// 64 (the third would spill: no gain).
template <typename T, int DT, int MQ, int BK, bool REST>
__global__ __launch_bounds__(256, DT > 64 || REST ? 2 : 3) void rel_attn_kernel(const RelAttn k) {
    typedef Dims<DT> Dm;
    constexpr bool WIDE = DT > 64;
    constexpr bool LEAN = REST && MQ * DT > 160;                            // two sets of accumulators: no registers for fragments read ahead
    constexpr int NB = BK / 16, VA = LEAN ? 0 : WIDE ? NB / 2 : 1, PT = pitch_of<T>(Dm::W);
    extern __shared__ __attribute__((aligned(32))) char lds[];
    const cv_rel_attn& a = k.a;
    T* tiles = reinterpret_cast<T*>(lds);                                    // K, V; K, V
    float* tab = reinterpret_cast<float*>(tiles + 4 * BK * PT);
    float* window = tab + k.G * a.num_buckets;

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g4 = lane >> 4, li = lane & 15;
    Part me;
    if (!part_of_block(k, me)) return;
    int tile = me.tile;
    const int split = me.split, kvh = me.kvh, s = me.s;
    if (a.q_off && a.zero_rest && tile + split + kvh == 0)
        zero_rest(a.q_off, s, a.n_seq, a.max_q, a.rows_q, reinterpret_cast<T*>(a.out), a.o_row, a.heads, a.o_head, a.head_dim);
    if (a.causal) tile = k.tiles - 1 - tile;                                 // the longest rows first
    const SeqRange qr = seq_range(a.q_off, s, a.max_q, a.rows_q), kr = seq_range(a.k_off, s, a.max_k, a.rows_k);
    const int rows = qr.len * k.G, r0 = tile * k.rt, q0 = tile * k.qt, shift = kr.len - qr.len, D = a.head_dim;
    if (r0 >= rows) return;
    const int rend = r0 + k.rt < rows ? r0 + k.rt : rows;
    const T* qb = reinterpret_cast<const T*>(a.q) + (a.q_off ? qr.row0 * a.q_row : s * a.q_seq) + (long)kvh * k.G * a.q_head;
    const T* kb = reinterpret_cast<const T*>(a.k) + (a.k_off ? kr.row0 * a.k_row : s * a.k_seq) + (long)kvh * a.k_head;
    const T* vb = reinterpret_cast<const T*>(a.v) + (a.k_off ? kr.row0 * a.v_row : s * a.v_seq) + (long)kvh * a.v_head;

    const int plo = q0 + shift, phi = (q0 + k.qt < qr.len ? q0 + k.qt : qr.len) - 1 + shift;       // positions of the tile
    int kend = kr.len;
    if (a.causal && phi + 1 < kend) kend = phi + 1 < 0 ? 0 : phi + 1;
    const int kbeg = split * k.split_tiles * BK;
    if (kend > kbeg + k.split_tiles * BK) kend = kbeg + k.split_tiles * BK;

    v8<T> qf[MQ][Dm::KS];
    int pos[MQ], head[MQ];
    float far_lo[MQ], far_hi[MQ];                                            // biases beyond the span, in exponents
    const bool busy = r0 + wave * MQ * 16 < rend;                            // a wave without rows only moves tiles
#pragma unroll
    for (int m = 0; m < MQ; ++m) {
        const int r = r0 + (wave * MQ + m) * 16 + li, qi = r / k.G;
        head[m] = r - qi * k.G;
        pos[m] = qi + shift;
        far_lo[m] = far_hi[m] = 0.f;
#pragma unroll
        for (int ks = 0; ks < Dm::KS; ++ks) qf[m][ks] = frag_global(qb + qi * a.q_row + head[m] * a.q_head, ks * 32 + g4 * 8, D, r < rend);
    }
    if (D < Dm::W) zero_pad_columns<T, Dm::W>(tiles, 4 * BK, PT, D);

    f32x4 o[MQ][Dm::ND], rest[REST ? MQ : 1][Dm::ND];
    float mref[MQ], l[MQ];                                                   // reference exponent (base 2), lane's part of the sum
#pragma unroll
    for (int m = 0; m < MQ; ++m) {
        mref[m] = NEG_INF; l[m] = 0.f;
#pragma unroll
        for (int d = 0; d < Dm::ND; ++d) {
            o[m][d] = (f32x4)(0.f);
            if constexpr (REST) rest[m][d] = (f32x4)(0.f);
        }
    }
    const int krb = (int)a.k_row * (int)sizeof(T), vrb = (int)a.v_row * (int)sizeof(T);
    Stage<T, BK, Dm::W> sk, sv;
    sk.init(krb, D, PT); sv.init(vrb, D, PT);
    int wbeg = 0, wend = 0;                                                  // offsets of the window
    // offsets a tile meets: k0 - phi .. k0 + BK - 1 - plo; near: some of them inside the span
    const int near_lo = plo - a.span - BK + 1, near_hi = a.table ? phi + a.span : near_lo;
    const auto near = [&](int k0) { return k0 > near_lo && k0 < near_hi; };
    const int whole = a.causal && plo + 1 < kr.len ? plo + 1 - BK : kr.len - BK;            // tiles up to here hide no key
    const auto window_for = [&](int k0) {                                    // before a barrier; every wave is past the last tile's products
        if (!near(k0) || k0 + BK - plo <= wend) return;
        __syncthreads();
        wbeg = k0 - phi; wend = wbeg + k.win;
        load_window(k, tab, k.G, window, wbeg);
    };
    const T *kp = kb + (long)kbeg * a.k_row, *vp = vb + (long)kbeg * a.v_row;
    const long kstep = (long)BK * a.k_row, vstep = (long)BK * a.v_row;
    if (kbeg < kend) {
        const int n = kr.len - kbeg < BK ? kr.len - kbeg : BK;
        sk.fetch(kp, n, krb, D); sv.fetch(vp, n, vrb, D);
        if (a.table) {
            load_table(k, kvh * k.G, k.G, tab);
            __syncthreads();
            const int blo = seq_bucket(a.map, a.span, a.num_buckets, -a.span), bhi = seq_bucket(a.map, a.span, a.num_buckets, a.span);
#pragma unroll
            for (int m = 0; m < MQ; ++m) { far_lo[m] = tab[head[m] * a.num_buckets + blo] * k.c; far_hi[m] = tab[head[m] * a.num_buckets + bhi] * k.c; }
            wend = kbeg - phi;                                               // nothing loaded
            window_for(kbeg);
        }
        sk.put(tiles); sv.put(tiles + BK * PT);
    }
#pragma unroll
    for (int m = 0; m < MQ; ++m)
#pragma unroll
        for (int ks = 0; ks < Dm::KS; ++ks) settle(qf[m][ks]);
    __syncthreads();
    int buf = 0;
    for (int k0 = kbeg; k0 < kend; k0 += BK) {
        const T* kt = tiles + buf * 2 * BK * PT;
        const T* vt = kt + BK * PT;
        const int next = k0 + BK;
        if (next < kend) {
            const int n = kr.len - next < BK ? kr.len - next : BK;
            kp += kstep; vp += vstep;
            sk.fetch(kp, n, krb, D);
            sv.fetch(vp, n, vrb, D);
        }
        if (busy) {
            f32x4 sc[NB][MQ];
            float bc[MQ];                                                    // bias of a far tile: one exponent a row
            v8<T> kf[NB][Dm::KS];
            const auto read_key = [&](int n, int ks) { return frag_row(kt + (n * 16 + li) * PT + ks * 32 + g4 * 8); };
            const auto key = [&](int n, int ks) { return LEAN ? read_key(n, ks) : kf[n][ks]; };
            if constexpr (!LEAN) {
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int ks = 0; ks < Dm::KS; ++ks) kf[n][ks] = read_key(n, ks);
            }
            if (near(k0)) {
#pragma unroll
                for (int m = 0; m < MQ; ++m) {
                    bc[m] = 0.f;
                    const int p = pos[m] <= phi ? pos[m] : phi;              // rows past the tile stay inside the window
                    const float* sp = reinterpret_cast<const float*>(lds) + whole_index((int)(window - reinterpret_cast<float*>(lds)) + head[m] * k.win + (k0 - wbeg - p) + 4 * g4);
#pragma unroll
                    for (int n = 0; n < NB; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r) sc[n][m][r] = sp[n * 16 + r];
                }
                if constexpr (WIDE && !LEAN) ahead<T>();
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int ks = 0; ks < Dm::KS; ++ks)
#pragma unroll
                        for (int m = 0; m < MQ; ++m) sc[n][m] = Seq<T>::mma(key(n, ks), qf[m][ks], sc[n][m]);
            } else {
                if constexpr (WIDE && !LEAN) ahead<T>();
#pragma unroll
                for (int m = 0; m < MQ; ++m) bc[m] = k0 >= phi ? far_hi[m] : far_lo[m];
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int ks = 0; ks < Dm::KS; ++ks)
#pragma unroll
                        for (int m = 0; m < MQ; ++m) sc[n][m] = Seq<T>::mma(key(n, ks), qf[m][ks], ks ? sc[n][m] : (f32x4)(0.f));
            }
            v8<T> vf[VA ? VA : 1][Dm::ND];                                   // on their way behind the exponentials
#pragma unroll
            for (int u = 0; u < VA; ++u)
#pragma unroll
                for (int d = 0; d < Dm::ND; ++d) vf[u][d] = frag_col(vt, PT, u * 32, d * 16, g4, li);
            if constexpr (!LEAN) ahead<T>();
            if (k0 > whole) {
#pragma unroll
                for (int m = 0; m < MQ; ++m) {
                    const int lim = (a.causal && pos[m] < kr.len - 1 ? pos[m] : kr.len - 1) - k0 - 4 * g4;
#pragma unroll
                    for (int n = 0; n < NB; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (n * 16 + r > lim) sc[n][m][r] = NEG_INF;
                }
            }
#pragma unroll
            for (int m = 0; m < MQ; ++m) {
                float mx = sc[0][m][0];
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) mx = max_of(mx, sc[n][m][r]);
                mx = fmaf(max_over_groups(mx), k.c, bc[m]);
                // The reference follows the maximum only when it is left behind by more than 2^8: p stays below 256, and the old sums are scaled
                // by the exact ratio of the references.
                if (__any(mx > mref[m] + 8.f)) {
                    const float up = mx > mref[m] ? mx : mref[m];
                    const float f = mref[m] == NEG_INF ? 0.f : exp2_hw(mref[m] - up);
                    mref[m] = up;
                    l[m] *= f;
#pragma unroll
                    for (int d = 0; d < Dm::ND; ++d) {
                        o[m][d] *= f;
                        if constexpr (REST) rest[m][d] *= f;
                    }
                }
                const float sub = bc[m] - (mref[m] == NEG_INF ? 0.f : mref[m]);
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int n = 0; n < NB; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float p = exp2_hw(fmaf(sc[n][m][r], k.c, sub));
                        sc[n][m][r] = p;
                        sum[r] += p;
                    }
                l[m] += (sum[0] + sum[1]) + (sum[2] + sum[3]);
            }
#pragma unroll
            for (int u = 0; u < NB / 2; ++u) {
                v8<T> pf[MQ], rf[REST ? Rest<T>::PARTS : 1][MQ];
#pragma unroll
                for (int m = 0; m < MQ; ++m) {
                    pf[m] = frag_acc<T>(sc[2 * u][m], sc[2 * u + 1][m]);     // p rounded to T once, for the product only
                    if constexpr (REST) {
#pragma unroll
                        for (int x = 0; x < Rest<T>::PARTS; ++x) rf[x][m] = next_part<T>(sc[2 * u][m], sc[2 * u + 1][m], x ? rf[x ? x - 1 : 0][m] : pf[m]);
                    }
                }
#pragma unroll
                for (int d = 0; d < Dm::ND; ++d) {
                    const v8<T> v = u < VA ? vf[u < VA ? u : 0][d] : frag_col(vt, PT, u * 32, d * 16, g4, li);
#pragma unroll
                    for (int m = 0; m < MQ; ++m) o[m][d] = mma_sum<T>(v, pf[m], o[m][d]);
                    if constexpr (REST) {
#pragma unroll
                        for (int x = 0; x < Rest<T>::PARTS; ++x)
#pragma unroll
                            for (int m = 0; m < MQ; ++m) rest[m][d] = Seq<T>::mma(v, rf[x][m], rest[m][d]);
                    }
                }
            }
        }
        if (next < kend) {
            buf ^= 1;
            sk.put(tiles + buf * 2 * BK * PT); sv.put(tiles + (buf * 2 + 1) * BK * PT);
            window_for(next);
        }
        __syncthreads();
    }
#pragma unroll
    for (int m = 0; m < MQ; ++m) {
        const int r = r0 + (wave * MQ + m) * 16 + li, qi = r / k.G;
        const float sum = sum_over_groups(l[m]);
        if (r >= rend) continue;
        const int h = kvh * k.G + head[m];
        const long row = (qr.row0 + qi) * a.heads + h;                       // [rows, heads]
        if (k.nsplit > 1) {
            const long pr = (((long)s * a.max_q + qi) * a.heads + h) * k.nsplit + split;
            if (g4 == 0) { k.part_ml[pr * 2] = mref[m]; k.part_ml[pr * 2 + 1] = sum; }
#pragma unroll
            for (int d = 0; d < Dm::ND; ++d)
                if (d * 16 + g4 * 4 < D) {
                    *reinterpret_cast<f32x4*>(k.part_o + pr * D + d * 16 + g4 * 4) = o[m][d];
                    if constexpr (REST) *reinterpret_cast<f32x4*>(k.part_rest + pr * D + d * 16 + g4 * 4) = rest[m][d];
                }
            continue;
        }
        const float inv = sum > 0.f ? 1.f / sum : sum == 0.f ? 0.f : sum;    // an empty row: zeros; NaN stays NaN
        if (a.lse && g4 == 0) a.lse[row] = sum > 0.f ? lse_of(mref[m], sum) : sum == 0.f ? NEG_INF : sum;
        T* ob = reinterpret_cast<T*>(a.out) + (a.q_off ? (qr.row0 + qi) * a.o_row : s * a.o_seq + qi * a.o_row) + h * a.o_head;
#pragma unroll
        for (int d = 0; d < Dm::ND; ++d) {
            const int c = d * 16 + g4 * 4;
            if (c >= D) continue;
            f32x4 x = o[m][d] * inv;
            settle(x);                                                       // one value for both: else the product is rounded to T at once in one of them
            store_rounded<T, 4>(ob + c, x);
            if (a.out_lo) store_rest<T>(a, row * D + c, x, REST ? rest[REST ? m : 0][d] * (inv / Rest<T>::UP) : (f32x4)(0.f));
        }
    }
}

// Up to 16 rows a key head (single tokens): one block of rows that all four waves share, each taking every fourth run of 32 keys, so nothing is
// waited for between waves until the end.  K goes from memory to registers as the product reads it, V through the wave's own piece of LDS (it is
// read transposed); the loads of a wave's next run are issued as soon as the registers of this one are free.  Bound by HBM: K and V once
// (16 ragged contexts to 32768, 4 key heads of 128, bf16: 116 us, 4.2 TB/s; 86 % of a copy's rate).
template <typename T, int DT, bool REST>
__global__ __launch_bounds__(256, sizeof(T) == 4 && DT > 96 ? 1 : 2) void rel_attn_few_kernel(const RelAttn k) {
    typedef Dims<DT> Dm;
    constexpr int KB = 32, PT = pitch_of<T>(Dm::W), E = 16 / sizeof(T), NV = KB * (Dm::W / E) / 64, HALVES = sizeof(T) / 2;
    extern __shared__ __attribute__((aligned(32))) char lds[];
    const cv_rel_attn& a = k.a;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g4 = lane >> 4, li = lane & 15;
    T* vt = reinterpret_cast<T*>(lds) + wave * KB * PT;
    float* tab = reinterpret_cast<float*>(reinterpret_cast<T*>(lds) + 4 * KB * PT);
    Part me;
    if (!part_of_block(k, me)) return;
    const int split = me.split, kvh = me.kvh, s = me.s;
    if (a.q_off && a.zero_rest && split + kvh == 0)
        zero_rest(a.q_off, s, a.n_seq, a.max_q, a.rows_q, reinterpret_cast<T*>(a.out), a.o_row, a.heads, a.o_head, a.head_dim);
    const SeqRange qr = seq_range(a.q_off, s, a.max_q, a.rows_q), kr = seq_range(a.k_off, s, a.max_k, a.rows_k);
    const int rows = qr.len * k.G, shift = kr.len - qr.len, D = a.head_dim;
    if (rows == 0) return;
    const T* qb = reinterpret_cast<const T*>(a.q) + (a.q_off ? qr.row0 * a.q_row : s * a.q_seq) + (long)kvh * k.G * a.q_head;
    const T* kb = reinterpret_cast<const T*>(a.k) + (a.k_off ? kr.row0 * a.k_row : s * a.k_seq) + (long)kvh * a.k_head;
    const T* vb = reinterpret_cast<const T*>(a.v) + (a.k_off ? kr.row0 * a.v_row : s * a.v_seq) + (long)kvh * a.v_head;
    const int plo = shift, phi = shift + qr.len - 1;
    int kend = kr.len;
    if (a.causal && phi + 1 < kend) kend = phi + 1 < 0 ? 0 : phi + 1;
    const int kbeg = split * k.split_tiles * KB;
    if (kend > kbeg + k.split_tiles * KB) kend = kbeg + k.split_tiles * KB;

    const int krb = (int)a.k_row * (int)sizeof(T), vrb = (int)a.v_row * (int)sizeof(T);
    u32x4 kn[2][Dm::KS][HALVES], vn[NV];                                     // the next run
    unsigned kat[2][Dm::KS], vat[NV];
    int vput[NV];
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int ks = 0; ks < Dm::KS; ++ks) kat[n][ks] = ks * 32 + g4 * 8 < D ? (unsigned)((n * 16 + li) * krb + (ks * 32 + g4 * 8) * (int)sizeof(T)) : 0xffffff00u;
    const int ppr = D / E;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int q = i * 64 + lane, r = q / ppr, col = (q - r * ppr) * E;
        vat[i] = r < KB ? (unsigned)(r * vrb + col * (int)sizeof(T)) : 0xffffff00u;
        vput[i] = r < KB ? r * PT + col : -1;
    }
    const auto range = [&](int k0, int rb) { const int n = kr.len - k0 < KB ? kr.len - k0 : KB; return (n - 1) * rb + D * (int)sizeof(T); };
    const auto fetch_k = [&](int k0) {
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(kb + (long)k0 * a.k_row), 0, range(k0, krb), 0x00027000);
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int ks = 0; ks < Dm::KS; ++ks)
#pragma unroll
                for (int x = 0; x < HALVES; ++x) kn[n][ks][x] = __builtin_amdgcn_raw_buffer_load_b128(rs, (int)kat[n][ks] + x * 16, 0, 0);
    };
    const auto fetch_v = [&](int k0) {
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(vb + (long)k0 * a.v_row), 0, range(k0, vrb), 0x00027000);
#pragma unroll
        for (int i = 0; i < NV; ++i) vn[i] = __builtin_amdgcn_raw_buffer_load_b128(rs, (int)vat[i], 0, 0);
    };
    const int first = kbeg + wave * KB;
    if (first < kend) { fetch_k(first); fetch_v(first); }

    v8<T> qf[Dm::KS];
    const int qi = li / k.G, head = li - qi * k.G, pos = qi + shift;
#pragma unroll
    for (int ks = 0; ks < Dm::KS; ++ks) qf[ks] = frag_global(qb + qi * a.q_row + head * a.q_head, ks * 32 + g4 * 8, D, li < rows);
    float far_lo = 0.f, far_hi = 0.f;
    if (a.table) {
        load_table(k, kvh * k.G, k.G, tab);
        __syncthreads();
        far_lo = tab[head * a.num_buckets + seq_bucket(a.map, a.span, a.num_buckets, -a.span)] * k.c;
        far_hi = tab[head * a.num_buckets + seq_bucket(a.map, a.span, a.num_buckets, a.span)] * k.c;
    }
    if (D < Dm::W) for (int r = lane; r < KB; r += 64) for (int c = D; c < Dm::W; c += E) store_piece(vt + r * PT + c, zero_piece());
    const int near_lo = plo - a.span - KB + 1, near_hi = a.table ? phi + a.span : near_lo;
    const int lim = a.causal && pos < kr.len - 1 ? pos : kr.len - 1;
    const int whole = a.causal && plo + 1 < kr.len ? plo + 1 - KB : kr.len - KB;

    f32x4 o[Dm::ND], rest[REST ? Dm::ND : 1];
#pragma unroll
    for (int d = 0; d < Dm::ND; ++d) {
        o[d] = (f32x4)(0.f);
        if constexpr (REST) rest[d] = (f32x4)(0.f);
    }
    float mref = NEG_INF, l = 0.f;
#pragma unroll
    for (int ks = 0; ks < Dm::KS; ++ks) settle(qf[ks]);
    for (int k0 = first; k0 < kend; k0 += 4 * KB) {
        f32x4 sc[2];
        float bc = 0.f;
        if (k0 > near_lo && k0 < near_hi) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    sc[n][r] = tab[head * a.num_buckets + seq_bucket(a.map, a.span, a.num_buckets, k0 + n * 16 + 4 * g4 + r - pos)];
        } else {
            bc = k0 >= phi ? far_hi : far_lo;
            sc[0] = sc[1] = (f32x4)(0.f);
        }
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int ks = 0; ks < Dm::KS; ++ks) sc[n] = Seq<T>::mma(__builtin_bit_cast(v8<T>, kn[n][ks]), qf[ks], sc[n]);
        const int next = k0 + 4 * KB;
        if (next < kend) fetch_k(next);
        if (k0 > whole) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (k0 + n * 16 + 4 * g4 + r > lim) sc[n][r] = NEG_INF;
        }
        float mx = max_of(max_of(max_of(sc[0][0], sc[0][1]), max_of(sc[0][2], sc[0][3])), max_of(max_of(sc[1][0], sc[1][1]), max_of(sc[1][2], sc[1][3])));
        mx = fmaf(max_over_groups(mx), k.c, bc);
        if (__any(mx > mref + 8.f)) {                                        // as in the kernel for many rows
            const float up = mx > mref ? mx : mref, f = mref == NEG_INF ? 0.f : exp2_hw(mref - up);
            mref = up;
            l *= f;
#pragma unroll
            for (int d = 0; d < Dm::ND; ++d) {
                o[d] *= f;
                if constexpr (REST) rest[d] *= f;
            }
        }
        const float sub = bc - (mref == NEG_INF ? 0.f : mref);
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) { sc[n][r] = exp2_hw(fmaf(sc[n][r], k.c, sub)); l += sc[n][r]; }
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (vput[i] >= 0) *reinterpret_cast<u32x4*>(vt + vput[i]) = vn[i];
        if (next < kend) fetch_v(next);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
        const v8<T> pf = frag_acc<T>(sc[0], sc[1]);
        v8<T> rf[REST ? Rest<T>::PARTS : 1];
        if constexpr (REST) {
#pragma unroll
            for (int x = 0; x < Rest<T>::PARTS; ++x) rf[x] = next_part<T>(sc[0], sc[1], x ? rf[x ? x - 1 : 0] : pf);
        }
#pragma unroll
        for (int d = 0; d < Dm::ND; ++d) {
            const v8<T> v = frag_col(vt, PT, 0, d * 16, g4, li);
            o[d] = mma_sum<T>(v, pf, o[d]);
            if constexpr (REST) {
#pragma unroll
                for (int x = 0; x < Rest<T>::PARTS; ++x) rest[d] = Seq<T>::mma(v, rf[x], rest[d]);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront", "local");
    }
    // join the waves: rows of D + 2 floats (sums, reference, weight), and the sums of what is left of P, in the space of V
    constexpr int RW = (REST ? 2 : 1) * DT + 4;
    float* join = reinterpret_cast<float*>(lds);
    const float sum = sum_over_groups(l);
    __syncthreads();
    float* mine = join + (wave * 16 + li) * RW;
#pragma unroll
    for (int d = 0; d < Dm::ND; ++d) {
        *reinterpret_cast<f32x4*>(mine + d * 16 + g4 * 4) = o[d];
        if constexpr (REST) *reinterpret_cast<f32x4*>(mine + DT + 4 + d * 16 + g4 * 4) = rest[d];
    }
    if (g4 == 0) { mine[DT] = mref; mine[DT + 1] = sum; }
    __syncthreads();
    // 16 threads a row, 4 columns a thread a turn
    const int row = threadIdx.x >> 4, qrow = row / k.G, h = kvh * k.G + row - qrow * k.G;
    if (row >= rows) return;
    float m[4], ref = NEG_INF, tot = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) { m[w] = join[(w * 16 + row) * RW + DT]; ref = fmaxf(ref, m[w]); }
#pragma unroll
    for (int w = 0; w < 4; ++w) { m[w] = exp2_hw(m[w] - (ref == NEG_INF ? 0.f : ref)); tot = fmaf(m[w], join[(w * 16 + row) * RW + DT + 1], tot); }
    const long out_row = (qr.row0 + qrow) * a.heads + h, pr = (((long)s * a.max_q + qrow) * a.heads + h) * k.nsplit + split;
    const float inv = tot > 0.f ? 1.f / tot : tot == 0.f ? 0.f : tot;
    if ((threadIdx.x & 15) == 0) {
        if (k.nsplit > 1) { k.part_ml[pr * 2] = ref; k.part_ml[pr * 2 + 1] = tot; }
        else if (a.lse) a.lse[out_row] = tot > 0.f ? lse_of(ref, tot) : tot == 0.f ? NEG_INF : tot;
    }
    T* ob = reinterpret_cast<T*>(a.out) + (a.q_off ? (qr.row0 + qrow) * a.o_row : s * a.o_seq + qrow * a.o_row) + h * a.o_head;
    for (int c = (threadIdx.x & 15) * 4; c < D; c += 64) {
        f32x4 v = (f32x4)(0.f), left = (f32x4)(0.f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            v += m[w] * *reinterpret_cast<const f32x4*>(join + (w * 16 + row) * RW + c);
            if constexpr (REST) left += m[w] * *reinterpret_cast<const f32x4*>(join + (w * 16 + row) * RW + DT + 4 + c);
        }
        if (k.nsplit > 1) {
            *reinterpret_cast<f32x4*>(k.part_o + pr * D + c) = v;
            if constexpr (REST) *reinterpret_cast<f32x4*>(k.part_rest + pr * D + c) = left;
            continue;
        }
        f32x4 x = v * inv;
        settle(x);                                                           // one value for both, as for many rows
        store_rounded<T, 4>(ob + c, x);
        if (a.out_lo) store_rest<T>(a, out_row * D + c, x, left * (inv / Rest<T>::UP));
    }
}

// Joins the key splits of a row: a wave a row, 16 lanes x 8 columns, four lanes of splits, in a fixed order (16 sequences x 16 heads, 32 splits: 9 us).
template <typename T, bool REST>
__global__ __launch_bounds__(256) void rel_attn_join_kernel(const RelAttn k) {
    const cv_rel_attn& a = k.a;
    const int lane = threadIdx.x & 63, c = (lane & 15) * 8, D = a.head_dim;
    const long pr = (long)blockIdx.x * 4 + (threadIdx.x >> 6);               // ((s * max_q) + qi) * heads + h
    if (pr >= (long)a.n_seq * a.max_q * a.heads) return;
    const int h = (int)(pr % a.heads);
    const long sq = pr / a.heads;
    const int qi = (int)(sq % a.max_q), s = (int)(sq / a.max_q);
    const SeqRange qr = seq_range(a.q_off, s, a.max_q, a.rows_q);
    if (qi >= qr.len) return;
    const float* ml = k.part_ml + pr * k.nsplit * 2;
    float top = NEG_INF;
    for (int i = lane; i < k.nsplit; i += 64) top = fmaxf(top, ml[i * 2]);
#pragma unroll
    for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
    const float ref = top == NEG_INF ? 0.f : top;
    float l = 0.f, o[8], left[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = left[j] = 0.f;
    const auto add = [&](float w, const float* src, float (&to)[8]) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(src), y = *reinterpret_cast<const f32x4*>(src + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) { to[j] = fmaf(w, x[j], to[j]); to[4 + j] = fmaf(w, y[j], to[4 + j]); }
    };
#pragma unroll 4
    for (int i = lane >> 4; i < k.nsplit; i += 4) {
        const float w = exp2_hw(ml[i * 2] - ref);
        l = fmaf(w, ml[i * 2 + 1], l);
        if (c < D) {
            add(w, k.part_o + (pr * k.nsplit + i) * D + c, o);
            if constexpr (REST) add(w, k.part_rest + (pr * k.nsplit + i) * D + c, left);
        }
    }
    l = sum_over_groups(l);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        o[j] = sum_over_groups(o[j]);
        if constexpr (REST) left[j] = sum_over_groups(left[j]);
    }
    const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
    if (a.lse && lane == 0) a.lse[(qr.row0 + qi) * a.heads + h] = l > 0.f ? lse_of(ref, l) : l == 0.f ? NEG_INF : l;
    if (lane >= 16 || c >= D) return;
    T* ob = reinterpret_cast<T*>(a.out) + (a.q_off ? (qr.row0 + qi) * a.o_row : s * a.o_seq + qi * a.o_row) + h * a.o_head + c;
#pragma unroll
    for (int j = 0; j < 8; ++j) { o[j] *= inv; settle(o[j]); left[j] *= inv / Rest<T>::UP; }
    store_rounded<T, 8>(ob, o);
    if (a.out_lo) {
        const long at = ((qr.row0 + qi) * a.heads + h) * D + c;
        store_rest<T>(a, at, f32x4{o[0], o[1], o[2], o[3]}, f32x4{left[0], left[1], left[2], left[3]});
        store_rest<T>(a, at + 4, f32x4{o[4], o[5], o[6], o[7]}, f32x4{left[4], left[5], left[6], left[7]});
    }
}

// keys a step: 64 (8 x 16 heads x 4096 x 80 fp16: 880 us, 912 with 32), or 32 where two buffers of 64 would leave little room for a second workgroup on a
// compute unit (heads of 128: dense 4 x 16 x 2048 204 us, 197 with 64; causal 8192 x 32 heads 639, 647; causal 2 x 577 33, 38)
constexpr int fwd_keys(bool wide, int D) { return wide || D > 96 ? 32 : 64; }

struct FwdPlan { int mq, rt, tiles, nsplit, split_tiles; };                  // mq 0: the kernel for few rows
// Up to 16 rows a key head: the kernel for few rows, keys split until there are about 2048 workgroups of 256 keys or more (fp16, one context of 32768 with 4
// key heads of 128: 31 us, 48 with the kernel for many rows; 8 of 2000: 13, 13; 64 of 4096: 105, 108; where there are many pairs the other is as
// good or better: 16 ragged to 32768 in bf16 116, 104; fp32 64 of 4096 231, 183).  Else 32 rows a wave with 16-bit types (K and V fragments serve two
// row blocks: 8 x 16 heads x 4096 x 80 880 us, 1186 with 16), 16 where that leaves less than two workgroups a compute unit (16 x 6 heads x
// 257 x 64: 12.2 us, 14.1 with 32); keys split when the row tiles alone leave compute units idle: until there are about 1024 workgroups, at
// least 4 key tiles each.
FwdPlan fwd_plan(const cv_rel_attn& a) {
    FwdPlan p;
    const int G = a.heads / a.kv_heads;
    const long rows = (long)a.max_q * G, pairs = (long)a.kv_heads * a.n_seq;
    int bk = 32, least = 8;
    long want = 2048;
    if (rows <= 16) { p.mq = 0; p.rt = 16 / G * G; p.tiles = 1; }
    else {
        p.mq = a.dtype != CV_DTYPE_F32 && pairs * ((rows + 127) / 128) >= 512 ? 2 : 1;
        p.rt = 64 * p.mq / G * G;
        p.tiles = (int)((rows + p.rt - 1) / p.rt);
        bk = fwd_keys(a.dtype == CV_DTYPE_F32, a.head_dim); least = 4; want = 1024;
    }
    const long base = p.tiles * pairs;
    const int key_tiles = (a.max_k + bk - 1) / bk;
    long n = base >= want / 2 ? 1 : want / base;
    if (n > key_tiles / least) n = key_tiles / least;
    if (n < 1) n = 1;
    p.split_tiles = (int)((key_tiles + n - 1) / n);
    if (p.mq == 0) p.split_tiles = (p.split_tiles + 3) & ~3;                 // the same number of runs for each of the four waves
    if (p.split_tiles < 1) p.split_tiles = 1;
    p.nsplit = (key_tiles + p.split_tiles - 1) / p.split_tiles;
    if (p.nsplit < 1) p.nsplit = 1;
    return p;
}

template <typename T, int DT, bool REST>
int few_launch(RelAttn& k, hipStream_t st) {
    const size_t v = 4 * 32 * pitch_of<T>(Dims<DT>::W) * sizeof(T) + (k.a.table ? (size_t)k.G * k.a.num_buckets * 4 : 0), join = 64 * ((REST ? 2 : 1) * DT + 4) * 4;
    const size_t bytes = v > join ? v : join;
    if (const int rc = allow_lds(&rel_attn_few_kernel<T, DT, REST>, bytes)) return rc;
    hipLaunchKernelGGL((rel_attn_few_kernel<T, DT, REST>), dim3(part_grid(k)), dim3(256), bytes, st, k);
    return (int)hipGetLastError();
}

template <typename T, int DT, int MQ, bool REST>
int fwd_launch(RelAttn& k, hipStream_t st) {
    constexpr int BK = fwd_keys(sizeof(T) == 4, DT);
    const int G = k.G;
    if (k.a.table) k.win = window_size(k.a, G, BK + 64 * MQ / G);
    const size_t bytes = 4 * BK * pitch_of<T>(Dims<DT>::W) * sizeof(T) + (k.a.table ? (size_t)G * (k.a.num_buckets + k.win) * 4 : 0);
    if (const int rc = allow_lds(&rel_attn_kernel<T, DT, MQ, BK, REST>, bytes)) return rc;
    hipLaunchKernelGGL((rel_attn_kernel<T, DT, MQ, BK, REST>), dim3(part_grid(k)), dim3(256), bytes, st, k);
    return (int)hipGetLastError();
}
template <typename T, int DT, int MQ> int fwd_pick(RelAttn& k, hipStream_t st) {
    if constexpr (sizeof(T) == 2)
        if (k.a.out_lo) {
            if constexpr (MQ == 0) return few_launch<T, DT, true>(k, st);
            else return fwd_launch<T, DT, MQ, true>(k, st);
        }
    if constexpr (MQ == 0) return few_launch<T, DT, false>(k, st);
    else return fwd_launch<T, DT, MQ, false>(k, st);
}
template <typename T, int MQ>
int fwd_dim(RelAttn& k, hipStream_t st) {
    const int D = k.a.head_dim;
    if (D <= 32) return fwd_pick<T, 32, MQ>(k, st);
    if (D <= 64) return fwd_pick<T, 64, MQ>(k, st);
    if (D <= 80) return fwd_pick<T, 80, MQ>(k, st);
    if (D <= 96) return fwd_pick<T, 96, MQ>(k, st);
    return fwd_pick<T, 128, MQ>(k, st);
}
template <typename T> int fwd_t(RelAttn& k, int mq, hipStream_t st) {
    int rc;
    if (mq == 0) rc = fwd_dim<T, 0>(k, st);
    else if constexpr (sizeof(T) == 2) rc = mq == 2 ? fwd_dim<T, 2>(k, st) : fwd_dim<T, 1>(k, st);
    else rc = fwd_dim<T, 1>(k, st);
    if (rc || k.nsplit == 1) return rc;
    const dim3 grid((unsigned)(((long)k.a.n_seq * k.a.max_q * k.a.heads + 3) / 4));
    bool rest = false;
    if constexpr (sizeof(T) == 2) {
        rest = k.a.out_lo != nullptr;
        if (rest) hipLaunchKernelGGL((rel_attn_join_kernel<T, true>), grid, dim3(256), 0, st, k);
    }
    if (!rest) hipLaunchKernelGGL((rel_attn_join_kernel<T, false>), grid, dim3(256), 0, st, k);
    return (int)hipGetLastError();
}

}  // namespace

// Rows of `heads` heads that no sequence owns because there are no sequences, or none of any length, so that no kernel starts that would zero them.  Moves
// 16 bytes a thread a turn.
__global__ __launch_bounds__(256) void rel_zero_kernel(char* base, long pieces, int per_row, int per_head, long row, long head) {
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < pieces; i += (long)gridDim.x * 256) {
        const long t = i / per_row;
        const int c = (int)(i - t * per_row), h = c / per_head;
        *reinterpret_cast<u32x4*>(base + t * row + h * head + (c - h * per_head) * 16) = u32x4{0u, 0u, 0u, 0u};
    }
}
int launch_rel_zero(void* base, int dtype, long rows, int heads, int D, long row, long head, hipStream_t st) {
    if (!base || rows <= 0) return 0;
    const int es = dtype == CV_DTYPE_F32 ? 4 : 2, per_head = D * es / 16;
    const long pieces = rows * heads * per_head, groups = (pieces + 255) / 256;
    hipLaunchKernelGGL(rel_zero_kernel, dim3((unsigned)(groups < 4096 ? groups : 4096)), dim3(256), 0, st, reinterpret_cast<char*>(base), pieces, heads * per_head, per_head, row * es,
                       head * es);
    return (int)hipGetLastError();
}

static bool keeps_rest(const cv_rel_attn& a) { return a.out_lo && a.dtype != CV_DTYPE_F32; }

int64_t rel_attention_tiles(const cv_rel_attn& a, bool grad) {
    if (grad) return rel_attention_bwd_tiles(a);
    if (a.n_seq == 0 || a.max_q == 0) return 0;
    const FwdPlan p = fwd_plan(a);
    return (int64_t)p.tiles * p.nsplit;
}
int64_t rel_attention_fwd_ws(const cv_rel_attn& a) {
    if (a.n_seq == 0 || a.max_q == 0) return 0;
    const FwdPlan p = fwd_plan(a);
    if (p.nsplit == 1) return 0;
    return (int64_t)a.n_seq * a.max_q * a.heads * p.nsplit * ((keeps_rest(a) ? 2 : 1) * a.head_dim + 2) * 4;
}

int launch_rel_attention(const cv_rel_attn& a, hipStream_t st) {
    if (a.n_seq == 0 || a.max_q == 0) return a.zero_rest && a.q_off ? launch_rel_zero(a.out, a.dtype, a.rows_q, a.heads, a.head_dim, a.o_row, a.o_head, st) : 0;
    const FwdPlan p = fwd_plan(a);
    RelAttn k{};
    k.a = a; k.G = a.heads / a.kv_heads; k.rt = p.rt; k.qt = p.rt / k.G; k.tiles = p.tiles; k.nsplit = p.nsplit; k.split_tiles = p.split_tiles;
    k.c = a.scale * LOG2E;
    if (!a.table) k.a.num_buckets = 0;
    k.part_o = reinterpret_cast<float*>(a.ws);
    const long rows = (long)a.n_seq * a.max_q * a.heads * p.nsplit;
    k.part_rest = k.part_o + rows * a.head_dim;
    k.part_ml = k.part_rest + (keeps_rest(a) ? rows * a.head_dim : 0);
    return a.dtype == CV_DTYPE_F16 ? fwd_t<half_t>(k, p.mq, st) : a.dtype == CV_DTYPE_BF16 ? fwd_t<bhalf_t>(k, p.mq, st) : fwd_t<float>(k, p.mq, st);
}

}  // namespace cva
