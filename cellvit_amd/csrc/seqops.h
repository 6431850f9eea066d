// Shared device helpers of the sequence operators (relbias.hip, relattn*.hip, blocknorm.hip).
#pragma once
#include "../../include/cellvit_amd.h"
#include "common.h"

void cva_set_error(const char* fmt, ...);

namespace cva {

typedef __bf16 bhalf_t;
typedef __bf16 bhalf8_t __attribute__((ext_vector_type(8)));

// Storage types of the sequence operators: fp16, bf16 (one 16x16x32 MFMA step per fragment) and fp32 (eight 16x16x4 steps).
template <typename T> struct Seq;
template <> struct Seq<half_t> {
    typedef half8_t vec8;
    static __device__ __forceinline__ f32x4 mma(const vec8& a, const vec8& b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <> struct Seq<bhalf_t> {
    typedef bhalf8_t vec8;
    static __device__ __forceinline__ f32x4 mma(const vec8& a, const vec8& b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Seq<float> {
    typedef float vec8 __attribute__((ext_vector_type(8)));
    // lane l holds k = (l >> 4) * 8 + j of both operands: step j contracts k in {j, 8 + j, 16 + j, 24 + j}
    static __device__ __forceinline__ f32x4 mma(const vec8& a, const vec8& b, f32x4 c) {
#pragma unroll
        for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
};

// c + a b for sums over many tiles.  fp32: the eight steps of a tile are summed by themselves first, so that a long sum is rounded once a tile at its full size
// instead of eight times (dV of 3600 rows: 1.2e-6 off, 6e-7 so); fp16 and bf16 have one step.
template <typename T> __device__ __forceinline__ f32x4 mma_sum(const typename Seq<T>::vec8& a, const typename Seq<T>::vec8& b, f32x4 c) {
    if constexpr (sizeof(T) == 4) return c + Seq<T>::mma(a, b, (f32x4)(0.f));
    else return Seq<T>::mma(a, b, c);
}

// Sum over the 64 lanes by row shifts and row broadcasts (no LDS): lane 63 holds it, readlane hands it to all.  Fixed order.
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float seq_wave_sum(float v) {
    v = dpp_add<0x111, 0xf>(v);      // row_shr:1
    v = dpp_add<0x112, 0xf>(v);      // row_shr:2
    v = dpp_add<0x114, 0xf>(v);      // row_shr:4
    v = dpp_add<0x118, 0xf>(v);      // row_shr:8  (lane 15 of a row: the row's sum)
    v = dpp_add<0x142, 0xa>(v);      // row_bcast:15 into rows 1 and 3
    v = dpp_add<0x143, 0xc>(v);      // row_bcast:31 into rows 2 and 3
    return __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(v), 63));
}

// Sums over the lanes by bucket in a fixed order: one pass per bucket present, lane (bucket & 63) of word bucket >> 6 receives its sum.
// All 64 lanes must call it; a lane without a value passes on = false.
__device__ __forceinline__ void seq_bucket_add(float v, int b, bool on, float (&acc)[4]) {
    const int lane = threadIdx.x & 63;
    unsigned long long todo = __ballot(on);
    while (todo) {
        const int bb = __builtin_amdgcn_readlane(b, __ffsll((unsigned long long)todo) - 1);
        const bool hit = on && b == bb;
        const float s = seq_wave_sum(hit ? v : 0.f);
        if ((bb & 63) == lane) {
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[r] += (bb >> 6) == r ? s : 0.f;
        }
        on = on && !hit;
        todo = __ballot(on);
    }
}

// The same for values whose buckets come in runs (neighbouring offsets): lane l holds the value of offset first + l, the sums are added to acc[bucket] in LDS,
// which no other wave touches.  A scan inside the runs leaves a run's sum in its last lane; the last lanes add them at once where a side's (offsets up to
// 0, above 0) buckets rise or fall throughout, so that no two meet, one after the other else.
__device__ __forceinline__ void seq_bucket_runs(float v, int b, bool on, int first, float* acc) {
    const int lane = threadIdx.x & 63;
    if (!on) { v = 0.f; b = -1; }
    const int before = __shfl_up(b, 1), after = __shfl_down(b, 1);
    const unsigned long long starts = __ballot(lane == 0 || b != before);
    const int start = 63 - __clzll(starts & (~0ull >> (63 - lane)));
#define SEQ_STEP(CTRL, ROWS, SRC) \
    do { \
        const float t = __uint_as_float((unsigned)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, ROWS, 0xf, false)); \
        v += start <= (SRC) ? t : 0.f; \
    } while (0)
    SEQ_STEP(0x111, 0xf, lane - 1);
    SEQ_STEP(0x112, 0xf, lane - 2);
    SEQ_STEP(0x114, 0xf, lane - 4);
    SEQ_STEP(0x118, 0xf, lane - 8);
    SEQ_STEP(0x142, 0xa, (lane & 48) - 1);
    SEQ_STEP(0x143, 0xc, 31);
#undef SEQ_STEP
    const bool last = on && (lane == 63 || b != after);
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        const bool mine = last && (side ? first + lane > 0 : first + lane <= 0);
        unsigned long long ends = __ballot(mine);
        if (!ends) continue;
        const bool pair = mine && lane < 63 && after >= 0 && (side || first + lane < 0);         // the next run is of this side, too
        if (!__any(pair && after > b) || !__any(pair && after < b)) {
            if (mine) acc[b] += v;
        } else {
            for (; ends; ends &= ends - 1) {
                const int l = __ffsll(ends) - 1, bb = __builtin_amdgcn_readlane(b, l);
                const float vv = __uint_as_float((unsigned)__builtin_amdgcn_readlane((int)__float_as_uint(v), l));
                if (lane == 0) acc[bb] += vv;
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

__device__ __forceinline__ int seq_clamp(int x, int lo, int hi) { return x < lo ? lo : (x > hi ? hi : x); }
// bucket of an offset; map entries outside the table are read as the nearest one inside
__device__ __forceinline__ int seq_bucket(const int32_t* __restrict__ map, int span, int nb, int off) {
    return seq_clamp(map[seq_clamp(off, -span, span) + span], 0, nb - 1);
}

// a table entry, a table gradient: fp32, or the call's own type
__device__ __forceinline__ float table_at(const void* t, int dtype, long i) {
    return dtype == CV_DTYPE_F32 ? reinterpret_cast<const float*>(t)[i] : dtype == CV_DTYPE_F16 ? (float)reinterpret_cast<const half_t*>(t)[i]
                                                                                               : (float)reinterpret_cast<const bhalf_t*>(t)[i];
}
__device__ __forceinline__ void table_set(void* t, int dtype, long i, float v) {
    if (dtype == CV_DTYPE_F32) reinterpret_cast<float*>(t)[i] = v;
    else if (dtype == CV_DTYPE_F16) reinterpret_cast<half_t*>(t)[i] = (half_t)v;
    else reinterpret_cast<bhalf_t*>(t)[i] = (bhalf_t)v;
}

int launch_rel_bias(int dtype, int tdtype, const void* table, const int32_t* map, int nb, int span, int heads, int q_len, int k_len, void* out, hipStream_t st);
int64_t rel_bias_grad_ws(int nb, int heads, int q_len, int k_len);
int launch_rel_bias_grad(int dtype, int tdtype, const void* dbias, const int32_t* map, int nb, int span, int batch, int heads, int q_len, int k_len, void* dtable,
                         float* ws, hipStream_t st);
int launch_block_norm(const cv_block_norm& a, hipStream_t st);
int64_t block_norm_grad_ws(const cv_block_norm& a);
int launch_block_norm_grad(const cv_block_norm& a, hipStream_t st);
int64_t rel_attention_tiles(const cv_rel_attn& a, bool grad);     // workgroups of the largest launch for one (sequence, key head) pair
int64_t rel_attention_fwd_ws(const cv_rel_attn& a);
int64_t rel_attention_bwd_ws(const cv_rel_attn& a);
int launch_rel_attention(const cv_rel_attn& a, hipStream_t st);
int launch_rel_attention_grad(const cv_rel_attn& a, hipStream_t st);

}  // namespace cva
