// Device parts shared by the forward and the backward of the attention with a bucketed position bias.
//
// Rows.  The query rows of one key head are packed as r = qi * G + g (G = heads / kv_heads query heads share the key head): a tile of rows covers
// neighbouring positions of all G heads, so K and V are read once for the group, a single token fills G rows of a tile, and a shared key
// head's gradient sums over its group inside one loop.
// A tile holds a whole number of positions.
// Tiles.  Every product is formed so that a lane owns 4 neighbouring rows of one column and the next product takes the accumulators as its operand as
// they lie (contraction index of lane group g4, element j: row 4 g4 + j of the first 16-row block, then of the second): forward and dQ
// hold S^T [key][query], dK / dV hold S [query][key].  The other operand comes transposed out of the row-major LDS tile.
#pragma once
#include "seqops.h"

namespace cva {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float BIAS_LIMIT = 1.6777216e7f;        // |bias| log2 e is held below 2^24: exp2's argument stays exact to 1 beyond any score
#define NEG_INF (-__builtin_inff())

struct RelAttn {                                  // kernel argument
    cv_rel_attn a;
    int G, tiles, nsplit, split_tiles;            // G query heads a key head; row (or key) tiles of a sequence; key splits and their key tiles
    int rt, qt;                                   // rows of a tile: the largest multiple of G it holds; its positions
    int ht;                                       // dQ: heads of a tile
    int spread;                                   // sequences of unknown lengths: deal (sequence, key head) pairs to the XCDs in turn
    int win;                                      // offsets of one head's bias window in LDS
    float c;                                      // scale * log2 e
    float* part_o; float* part_rest; float* part_ml;       // partial results of the splits
    float* delta;                                 // backward: (lse, +inf where a row saw no key; rowsum(dout * out)) of the rows
    int* row_exp; float* amax; int n_amax;        // fp16's backward: exponents of the rows' dS; max |v_j|^2 of a (sequence, key head) pair in n_amax parts
    float* dpart; int units;                      // backward: partial table gradients
};

struct SeqRange { long row0; int len; };          // first packed row (dense: s * max) and length
__device__ __forceinline__ SeqRange seq_range(const int32_t* off, int s, int most, long rows) {
    SeqRange r;
    if (!off) { r.row0 = (long)s * most; r.len = most; return r; }
    long b = off[s], e = off[s + 1];              // ranges outside the rows are cut: a bad offset never leads outside the buffers
    b = b < 0 ? 0 : (b > rows ? rows : b);
    e = e < b ? b : (e > rows ? rows : e);
    r.row0 = b; r.len = (int)(e - b < most ? e - b : most);
    return r;
}

// A workgroup's part: tile, key split, key head, sequence.  The tiles of one (sequence, key head) pair run on one XCD, whose L2 (and address translation:
// splits of single tokens share nothing else, and lose 10 % when dealt as they come) then serves its K and V.  XCDs get equal runs of
// workgroups, or, with lengths known on the device only, pairs in turn, starting one further each round (a run would give one XCD the
// long sequences, rounds that start alike the same sequences' heads).
struct Part { int tile, split, kvh, s; };
__device__ __forceinline__ bool part_of_block(const RelAttn& k, Part& p) {
    const int per = k.tiles * k.nsplit;
    int pair, rest;
    if (k.spread) {
        const int i = blockIdx.x >> 3, turn = i / per;
        pair = turn * 8 + ((blockIdx.x - turn) & 7); rest = i - turn * per;
        if (pair >= k.a.kv_heads * k.a.n_seq) return false;
    } else {
        const int id = xcd_remap(blockIdx.x, gridDim.x);
        pair = id / per; rest = id - pair * per;
    }
    p.split = rest / k.tiles; p.tile = rest - p.split * k.tiles;
    p.s = pair / k.a.kv_heads; p.kvh = pair - p.s * k.a.kv_heads;
    return true;
}
inline unsigned part_grid(RelAttn& k) {
    const long pairs = (long)k.a.kv_heads * k.a.n_seq;
    k.spread = (k.a.q_off || k.a.k_off) && pairs >= 16;
    return (unsigned)((k.spread ? (pairs + 7) / 8 * 8 : pairs) * k.tiles * k.nsplit);
}

// Rows that no sequence owns: what sequence s was cut by, before the first, behind the last.  One workgroup a sequence zeroes them.
template <typename T>
__device__ __forceinline__ void zero_rest(const int32_t* off, int s, int n_seq, int most, long rows, T* base, long row, int heads, long head, int D) {
    const SeqRange r = seq_range(off, s, most, rows);
    const auto fill = [&](long a, long b) {
        const int ppr = heads * D * (int)sizeof(T) / 16;                  // 16-byte pieces of a row's heads
        for (long i = threadIdx.x; i < (b - a) * ppr; i += 256) {
            const long t = i / ppr;
            const int c = (int)(i - t * ppr) * (16 / (int)sizeof(T)), h = c / D;
            store_piece(base + (a + t) * row + h * head + (c - h * D), zero_piece());
        }
    };
    long e = off[s + 1];
    e = e < r.row0 ? r.row0 : (e > rows ? rows : e);
    fill(r.row0 + r.len, s == n_seq - 1 ? rows : e);
    if (s == 0) fill(0, r.row0);
}

template <int DT> struct Dims {
    static constexpr int KS = (DT + 31) / 32, ND = DT / 16, W = KS * 32;      // contraction steps over the head dimension, 16-wide blocks of it, LDS row
};
template <typename T> __host__ __device__ constexpr int pitch_of(int w) { return w + 32 / (int)sizeof(T); }   // elements; rows 32 B apart in the banks

template <typename T> using v8 = typename Seq<T>::vec8;
template <typename T> __device__ __forceinline__ v8<T> frag_row(const T* p) { return *reinterpret_cast<const v8<T>*>(p); }
template <typename T> __device__ __forceinline__ v8<T> frag_zero() {
    v8<T> f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (T)0.f;
    return f;
}
// 8 elements of a row in global memory, columns from D on read as 0 (D % 8 == 0)
template <typename T> __device__ __forceinline__ v8<T> frag_global(const T* row, int col, int D, bool on) {
    return on && col < D ? *reinterpret_cast<const v8<T>*>(row + col) : frag_zero<T>();
}
// A fragment that stays in registers: its loads are waited for here.  Without this the wait sits at the first product of the tile loop, where it would hold up
// the next tile's loads in every turn.
template <typename V> __device__ __forceinline__ void settle(V& f) {
    typedef unsigned words __attribute__((ext_vector_type(sizeof(V) / 4)));
    words w = __builtin_bit_cast(words, f);
    asm volatile("" : "+v"(w));
    f = __builtin_bit_cast(V, w);
}
// An index into LDS whose constant part stays in it: folded into each read's address it would not fit the paired reads' offsets, and every read would
// get an addition of its own.
__device__ __forceinline__ int whole_index(int i) { asm("" : "+v"(i)); return i; }
__device__ __forceinline__ void settle(float& f) { asm volatile("" : "+v"(f)); }
// A operand X^T[d0 + li][rows of the pair of 16-row blocks at r0]: element j = X[r0 + 4 g + j][d0 + li], j + 4: sixteen rows further
template <typename T> __device__ __forceinline__ v8<T> frag_col(const T* tile, int pitch, int r0, int d0, int g, int li) {
    v8<T> f;
    if constexpr (sizeof(T) == 2) {
        typedef short s4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s4* lds4;
        const T* p = tile + (r0 + 4 * g + (li >> 2)) * pitch + d0 + 4 * (li & 3);
        union { s4 h[2]; v8<T> v; } u;
        u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p));
        u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + 16 * pitch));
        f = u.v;
    } else {
        const T* p = tile + (r0 + 4 * g) * pitch + d0 + li;
#pragma unroll
        for (int j = 0; j < 4; ++j) { f[j] = p[j * pitch]; f[4 + j] = p[(16 + j) * pitch]; }
    }
    return f;
}
// LDS reads above stay above: left to itself the compiler reads each fragment right before its product and every product waits.  (fp32 fragments are twice
// as long: no registers for that.)
template <typename T> __device__ __forceinline__ void ahead() {
    if constexpr (sizeof(T) == 2) __builtin_amdgcn_sched_barrier(0);
}
template <typename T> __device__ __forceinline__ v8<T> frag_acc(const f32x4& a, const f32x4& b) {
    v8<T> f;
#pragma unroll
    for (int j = 0; j < 4; ++j) { f[j] = (T)a[j]; f[4 + j] = (T)b[j]; }
    return f;
}

// Stages ROWS rows of a matrix through registers into LDS in 16-byte pieces.  What a thread moves is the same in every tile, so its offsets are computed
// once; fetch() issues the loads of a tile through a buffer descriptor whose range ends behind row n - 1: later rows read as 0.
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
template <typename T, int ROWS, int W>
struct Stage {
    static constexpr int E = 16 / sizeof(T);                       // elements of a piece
    static constexpr int N = (ROWS * (W / E) + 255) / 256;         // pieces a thread at most
    u32x4 p[N];
    unsigned at[N]; int lds[N];                                    // byte offset in the tile's memory; element offset in LDS
    // no piece: the columns behind the row, that no product reads (a test would cost more than the write)
    static __device__ __forceinline__ int spare(int pitch) { return ((int)threadIdx.x % ROWS) * pitch + W; }
    __device__ __forceinline__ void init(int row_bytes, int D, int pitch) {
        const int ppr = D / E;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int q = i * 256 + threadIdx.x, r = q / ppr, col = (q - r * ppr) * E;
            at[i] = r < ROWS ? (unsigned)(r * row_bytes + col * (int)sizeof(T)) : 0xffffffffu;
            lds[i] = r < ROWS ? r * pitch + col : spare(pitch);
        }
    }
    // rows packed as position * G + head, of a tile of `rt` rows
    __device__ __forceinline__ void init_rows(int row_bytes, int head_bytes, int G, int rt, int D, int pitch) {
        const int ppr = D / E;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int q = i * 256 + threadIdx.x, r = q / ppr, col = (q - r * ppr) * E, qi = r / G;
            at[i] = r < rt ? (unsigned)(qi * row_bytes + (r - qi * G) * head_bytes + col * (int)sizeof(T)) : 0xffffffffu;
            lds[i] = r < ROWS ? r * pitch + col : spare(pitch);    // rows rt .. ROWS - 1 hold 0
        }
    }
    __device__ __forceinline__ void fetch(const T* base, int n, int row_bytes, int D) {
        const int range = n > 0 ? (n - 1) * row_bytes + D * (int)sizeof(T) : 0;
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), 0, range, 0x00027000);
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = __builtin_amdgcn_raw_buffer_load_b128(rs, (int)at[i], 0, 0);
    }
    // n rows of the tile are there (rows may lie in any order in memory, so the range does not end them)
    __device__ __forceinline__ void fetch_rows(const T* base, int n, int pitch) {
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), 0, 0x7fffffff, 0x00027000);
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = __builtin_amdgcn_raw_buffer_load_b128(rs, lds[i] < n * pitch ? (int)at[i] : -1, 0, 0);
    }
    __device__ __forceinline__ void put(T* tile) const {
#pragma unroll
        for (int i = 0; i < N; ++i)
            *reinterpret_cast<u32x4*>(tile + lds[i]) = p[i];
    }
};
// columns D .. W - 1 of n rows
template <typename T, int W> __device__ __forceinline__ void zero_pad_columns(T* rows, int n, int pitch, int D) {
    for (int r = threadIdx.x; r < n; r += 256)
        for (int c = D; c < W; c += 16 / (int)sizeof(T)) store_piece(rows + r * pitch + c, zero_piece());
}

// The bias of one head group in accumulator units (bias / scale: it is the products' starting value, so it costs no instruction).  A finite bias stays
// finite; -inf hides the key.
__device__ __forceinline__ float bias_unit(float b, float scale) {
    const float lim = BIAS_LIMIT / LOG2E;
    if (b > lim) b = b == __builtin_inff() ? b : lim;
    if (b < -lim) b = b == NEG_INF ? b : -lim;
    return b / scale;
}
// n heads from head h0 on
__device__ __forceinline__ void load_table(const RelAttn& k, int h0, int n, float* tab) {
    const cv_rel_attn& a = k.a;
    for (int i = threadIdx.x; i < n * a.num_buckets; i += 256) {
        const int g = i / a.num_buckets, b = i - g * a.num_buckets;
        tab[i] = bias_unit(table_at(a.table, a.table_dtype, (long)b * a.heads + h0 + g), a.scale);
    }
}
// The window: bias of n heads at offsets beg .. beg + win - 1, in LDS.  A tile of keys and rows meets keys + positions - 1 neighbouring
// offsets; the window is loaded again when a tile's run past its end (for a short span: once).
__device__ __forceinline__ void load_window(const RelAttn& k, const float* tab, int n, float* window, int beg, uint8_t* buckets = nullptr) {
    const cv_rel_attn& a = k.a;
    for (int x = threadIdx.x; x < k.win; x += 256) {
        const int b = seq_bucket(a.map, a.span, a.num_buckets, beg + x);
        if (buckets) buckets[x] = (uint8_t)b;
        for (int g = 0; g < n; ++g) window[g * k.win + x] = tab[g * a.num_buckets + b];
    }
}
// offsets of a window: all that are not saturated and a tile's run on either side where that is little, at least one tile's run
inline int window_size(const cv_rel_attn& a, int G, int run) {
    int w = 2 * a.span + 2 * run, most = 2048 / G;
    const long all = (long)a.max_k + a.max_q + run;                    // offsets there can be
    if (w > all) w = (int)all;
    if (w > most) w = most;
    return ((w < run ? run : w) + 3) & ~3;
}

// more than 64 KB of LDS has to be asked for, kernel by kernel (a workgroup may hold 160 KB, a few words of them static)
template <typename F> inline int allow_lds(F* kernel, size_t bytes) {
    if (bytes <= 65000) return 0;
    if (bytes > 163840 - 64) return (int)hipErrorInvalidValue;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != hipSuccess) (void)hipGetLastError();
    return (int)e;
}

int64_t rel_attention_bwd_tiles(const cv_rel_attn& a);
int launch_rel_zero(void* base, int dtype, long rows, int heads, int D, long row, long head, hipStream_t st);

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
// ref + log2(sum) rounded once: the sum's exponent is added exactly, so the logarithm that the hardware rounds is one of 1/2 .. 1.  (Of the whole sum it is off by
// a step of 8 or more, towards below on average, and the backward's P of the row with it.)
__device__ __forceinline__ float lse_of(float ref, float sum) {
    const float e = (float)__builtin_amdgcn_frexp_expf(sum), s = ref + e, part = s - ref;
    const float lost = (ref - (s - part)) + (e - part);
    return s + (lost + __builtin_amdgcn_logf(__builtin_amdgcn_frexp_mantf(sum)));
}
// four or eight neighbouring results, rounded
template <typename T, int N, typename V> __device__ __forceinline__ void store_rounded(T* dst, const V& x) {
    typedef T tn __attribute__((ext_vector_type(N)));
    tn v;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = (T)x[j];
    *reinterpret_cast<tn*>(dst) = v;
}
// What rounding took from four neighbouring results that end up as x: their own last one, and `rest` that the rounding of P had taken before
template <typename T, typename V> __device__ __forceinline__ void store_rest(const cv_rel_attn& a, long at, const V& x, const f32x4& rest) {
    typedef T t4 __attribute__((ext_vector_type(4)));
    f32x4 lo;
#pragma unroll
    for (int j = 0; j < 4; ++j) lo[j] = (x[j] - (float)(T)x[j]) + rest[j];
    if (a.lo_f32) { *reinterpret_cast<f32x4*>(reinterpret_cast<float*>(a.out_lo) + at) = lo; return; }
    t4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = (T)lo[j];
    *reinterpret_cast<t4*>(reinterpret_cast<T*>(a.out_lo) + at) = v;
}
// P for the product with V is rounded to T.  The backward's D = rowsum(dout out) goes into every dS of a row, so what that rounding takes from a row moves all of
// them one way, and a bucket of the table's gradient collects it from its rows: 2e-4 (fp16) to 2e-3 (bf16) of a table's gradient at 1500 keys.  A forward
// that is asked for `out_lo` (REST) sums what is left of P, too, in accumulators of its own, so that `out` keeps its bits: one more part of 11 bits in fp16, on
// a scale of 2^12 (above the subnormals), two of 8 bits in bf16 (one would leave 1e-6 .. 6e-6).  Then the table's gradient is good to fp32.
template <typename T> struct Rest;
template <> struct Rest<half_t> { static constexpr int PARTS = 1; static constexpr float UP = 4096.f; };
template <> struct Rest<bhalf_t> { static constexpr int PARTS = 2; static constexpr float UP = 1.f; };
template <> struct Rest<float> { static constexpr int PARTS = 0; static constexpr float UP = 1.f; };
// the next part of what is left of a block of P; `part`: the one taken last (UP is 1 where there is more than one)
template <typename T> __device__ __forceinline__ v8<T> next_part(f32x4& a, f32x4& b, const v8<T>& part) {
    v8<T> f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        a[j] -= (float)part[j]; b[j] -= (float)part[4 + j];
        f[j] = (T)(a[j] * Rest<T>::UP); f[4 + j] = (T)(b[j] * Rest<T>::UP);
    }
    return f;
}

// The four lane groups (lanes 16 g4 .. 16 g4 + 15) hold parts of one column: their maximum / sum, in every lane.  The swaps exchange rows of 16, then
// halves, between two registers (here twice the same), at the cost of a move; a shuffle through LDS would stand in every tile's way.
__device__ __forceinline__ void other_groups(float v, float& a, float& b, bool half) {
    const unsigned u = __float_as_uint(v);
    const auto r = half ? __builtin_amdgcn_permlane32_swap(u, u, false, false) : __builtin_amdgcn_permlane16_swap(u, u, false, false);
    a = __uint_as_float(r[0]); b = __uint_as_float(r[1]);
}
// NaN wins (fmaxf costs an instruction more an operand, to make it lose): a row with a NaN score is NaN either way
__device__ __forceinline__ float max_of(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float max_over_groups(float v) {
    float a, b;
    other_groups(v, a, b, false); v = max_of(a, b);
    other_groups(v, a, b, true); return max_of(a, b);
}
__device__ __forceinline__ float sum_over_groups(float v) {
    float a, b;
    other_groups(v, a, b, false); v = a + b;
    other_groups(v, a, b, true); return a + b;
}

}  // namespace cva
