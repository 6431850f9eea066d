// The learned position bias by buckets as a plane, and its gradient.
//   B[h, i, j] = t[map(j - i - shift), h],  shift = Lk - Lq           dt[c, h] = sum over s, i, j with map(..) = c of dB[s, h, i, j]
// Both are bound by HBM: the plane is written once (H Lq Lk elements), its gradient read once; tables and maps stay in cache.
#include <type_traits>

#include "seqops.h"

namespace cva {
namespace {

constexpr int BIAS_ITER = 4;                      // 16-byte groups a thread writes
constexpr int BIAS_CHUNK = 256 * 8 * BIAS_ITER;   // elements of a workgroup

// One workgroup writes a run of the flat plane of one head in 16-byte stores aligned in the whole output (Lk may be odd, so rows are not aligned); a
// group that straddles two heads is written by both, element by element, each its own part.  A group inside one row whose offsets all lie
// beyond the span is one value and needs no map (most of a long plane).  16 x 2048 x 4097 bf16: 48 us, 5.6 TB/s (a fill reaches 6.8).
template <typename T, int VEC>
__global__ __launch_bounds__(256) void rel_bias_kernel(const void* __restrict__ table, int tdtype, const int32_t* __restrict__ map, int nb, int span, int heads,
                                                       int q_len, int k_len, T* __restrict__ out) {
    typedef T vec_t __attribute__((ext_vector_type(VEC)));
    __shared__ float tab[256];
    const int h = blockIdx.y;
    for (int b = threadIdx.x; b < nb; b += 256) tab[b] = table_at(table, tdtype, (long)b * heads + h);
    __syncthreads();
    const long plane = (long)q_len * k_len, first = (long)h * plane;
    const long g0 = first / VEC + (long)blockIdx.x * (256 * BIAS_ITER);
    // row and column of the first element of this workgroup; the rest follows from 32-bit divisions relative to it
    const long p0 = g0 * VEC - first;                                   // may be negative in the first workgroup
    const long i0 = p0 < 0 ? 0 : p0 / k_len;
    const int j0 = (int)(p0 - i0 * k_len);                              // >= -VEC
    const int shift = k_len - q_len;
    const float low = tab[seq_bucket(map, span, nb, -span)], high = tab[seq_bucket(map, span, nb, span)];
#pragma unroll
    for (int it = 0; it < BIAS_ITER; ++it) {
        const int local = (it * 256 + (int)threadIdx.x) * VEC;
        const long p = p0 + local;
        if (p >= plane) return;
        const unsigned jj = (unsigned)(j0 + local < 0 ? 0 : j0 + local);
        const unsigned di = jj / (unsigned)k_len;
        long i = i0 + di;
        int j = j0 + local < 0 ? j0 + local : (int)(jj - di * (unsigned)k_len);
        T v[VEC];
        const int o = j - (int)i - shift;
        if (j >= 0 && j + VEC <= k_len && (o >= span || o + VEC - 1 <= -span)) {
            const T c = (T)(o >= span ? high : low);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = c;
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                v[e] = (T)tab[seq_bucket(map, span, nb, j - (int)i - shift)];
                if (++j == k_len) { j = 0; ++i; }
            }
        }
        T* dst = out + (g0 * VEC + local);
        if (p >= 0 && p + VEC <= plane) {
            vec_t w;
#pragma unroll
            for (int e = 0; e < VEC; ++e) w[e] = v[e];
            *reinterpret_cast<vec_t*>(dst) = w;
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (p + e >= 0 && p + e < plane) dst[e] = v[e];
        }
    }
}

// A lane follows VEC neighbouring diagonals down a band of rows and through the batch: all pairs of a diagonal share an offset, so the sums stay in
// registers and the map is read once a lane.  The loads run with the row (address + k_len + 1 a row): a wave reads 64 VEC contiguous elements.  At the end the
// wave adds its diagonals by bucket and writes one row of partial sums; rel_bias_reduce_kernel adds those.  2 x 16 x 2048 x 4097 bf16: 152 us, 3.5 TB/s;
// rows of odd length take a fifth 4-byte load and a shift (255 us with 16-byte loads at odd elements).
constexpr int GRAD_ROWS = 128;                     // rows of a band

template <typename T, int VEC>
__global__ __launch_bounds__(256) void rel_bias_grad_kernel(const T* __restrict__ dbias, const int32_t* __restrict__ map, int nb, int span, int batch,
                                                            int heads, int q_len, int k_len, int units, float* __restrict__ part) {
    typedef unsigned u4 __attribute__((ext_vector_type(4), aligned(4)));
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = blockIdx.z;
    const int r0 = blockIdx.y * GRAD_ROWS, r1 = r0 + GRAD_ROWS < q_len ? r0 + GRAD_ROWS : q_len;
    // column of the lane's first diagonal in row r0; the band touches columns-in-row-r0 from -(GRAD_ROWS - 1) to k_len - 1
    const int w0 = ((blockIdx.x * 4 + wave) * 64) * VEC - (GRAD_ROWS - 1), c0 = w0 + lane * VEC;
    // A plane's part of a diagonal is a run of up to GRAD_ROWS additions; the runs of a batch are added with what each addition took (rows of one sign would
    // lose 6e-5 of a batch of 64 in one run of 8192).
    float acc[VEC], total_of[VEC], took[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = total_of[e] = took[e] = 0.f;
    const long plane = (long)q_len * k_len, total = (long)batch * heads * plane;
    // Eight rows of loads are in flight.  16-byte loads at an odd 16-bit element are taken apart by the memory pipe, so such a row (its parity is the same in
    // all lanes) is read from the element before and shifted.  Only a wave at the plane's ends tests: a lane that reaches over a row's end
    // reads into the neighbouring row and drops what is not its own.
    const auto band = [&](auto edge) {
        constexpr bool EDGE = decltype(edge)::value;
        for (int s = 0; s < batch; ++s) {
            const long at0 = ((long)s * heads + h) * plane + (long)r0 * k_len + c0;
            const T* p0 = dbias + at0;
            for (int r = 0; r < r1 - r0; r += 8, p0 += 8 * (long)(k_len + 1)) {
                u4 x[8];
                unsigned more[8];
                bool odd[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const T* p = p0 + u * (long)(k_len + 1);
                    odd[u] = sizeof(T) == 2 && __builtin_amdgcn_readfirstlane((int)((uintptr_t)p & 2)) != 0;
                    const unsigned* q = reinterpret_cast<const unsigned*>((uintptr_t)p & ~(uintptr_t)3);
                    more[u] = 0u;
                    if constexpr (EDGE) {
                        const long at = at0 + (long)(r + u) * (k_len + 1);
                        const int c = c0 + r + u;
                        const bool on = c + VEC > 0 && c < k_len && r0 + r + u < r1;
                        x[u] = u4{0u, 0u, 0u, 0u};
                        if (at - 1 >= 0 && at + VEC + 1 <= total) {
                            if (on) { x[u] = *reinterpret_cast<const u4*>(q); if (odd[u]) more[u] = q[4]; }
                        } else if (on) {                                     // the tensor's first and last elements: nothing lies beyond them
#pragma unroll
                            for (int e = 0; e < VEC; ++e)
                                if (c + e >= 0 && c + e < k_len) acc[e] += (float)p[e];
                        }
                    } else {
                        x[u] = *reinterpret_cast<const u4*>(q);
                        if (odd[u] && lane == 63) more[u] = q[4];            // the other lanes take their right neighbour's first word
                    }
                }
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    float v[VEC];
                    if constexpr (sizeof(T) == 2) {
                        typedef T t2 __attribute__((ext_vector_type(2)));
                        if (odd[u]) {
                            if constexpr (!EDGE) more[u] = (unsigned)__builtin_amdgcn_update_dpp((int)more[u], (int)x[u][0], 0x130, 0xf, 0xf, false);      // wave_shl:1
#pragma unroll
                            for (int d = 0; d < 4; ++d) x[u][d] = __builtin_amdgcn_alignbit(d < 3 ? x[u][d + 1] : more[u], x[u][d], 16);
                        }
#pragma unroll
                        for (int d = 0; d < 4; ++d) {
                            const unsigned word = x[u][d];
                            const t2 w = __builtin_bit_cast(t2, word);
                            v[2 * d] = (float)w[0]; v[2 * d + 1] = (float)w[1];
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < VEC; ++e) v[e] = __uint_as_float(x[u][e]);
                    }
#pragma unroll
                    for (int e = 0; e < VEC; ++e) {
                        const int c = c0 + r + u + e;
                        acc[e] += !EDGE || (c >= 0 && c < k_len) ? v[e] : 0.f;
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float y = acc[e] - took[e], t = total_of[e] + y;
                took[e] = (t - total_of[e]) - y;
                total_of[e] = t;
                acc[e] = 0.f;
            }
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] = total_of[e];
    };
    // the last element of the tensor has no neighbour to be read with it: those waves test, too
    if (w0 >= 1 && w0 + 64 * VEC + GRAD_ROWS < k_len && r1 - r0 == GRAD_ROWS) band(std::false_type{});
    else band(std::true_type{});
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    const int base = c0 - r0 - (k_len - q_len);
    const bool on = c0 < k_len;                   // diagonals behind the plane's last hold nothing
    if (__all(!on || base >= span) || __all(!on || base + VEC - 1 <= -span)) {      // one bucket for the whole wave
        float v = 0.f;
#pragma unroll
        for (int e = 0; e < VEC; ++e) v += acc[e];
        seq_bucket_add(v, seq_bucket(map, span, nb, base), on, sum);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) seq_bucket_add(acc[e], seq_bucket(map, span, nb, base + e), on, sum);
    }
    float* dst = part + (((long)h * units) + (blockIdx.y * gridDim.x + blockIdx.x) * 4 + wave) * nb;
#pragma unroll
    for (int r = 0; r < 4; ++r)
        if (r * 64 + lane < nb) dst[r * 64 + lane] = sum[r];
}

// dtable[b, h] = sum over units of part[h, unit, b]: one workgroup per (64 buckets, head), 16 unit lanes x 64 buckets, joined in LDS in a fixed order
__global__ __launch_bounds__(1024) void rel_bias_reduce_kernel(const float* __restrict__ part, int units, int nb, int heads, void* __restrict__ dtable, int tdtype) {
    __shared__ float red[16][64];
    const int h = blockIdx.y, b = blockIdx.x * 64 + (threadIdx.x & 63), u0 = threadIdx.x >> 6;
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    if (b < nb) {
        const float* src = part + (long)h * units * nb + b;
        int u = u0;
        for (; u + 48 < units; u += 64) {
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[k] += src[(long)(u + 16 * k) * nb];
        }
        for (; u < units; u += 16) acc[0] += src[(long)u * nb];
    }
    red[u0][threadIdx.x & 63] = (acc[0] + acc[1]) + (acc[2] + acc[3]);
    __syncthreads();
    if (u0 == 0 && b < nb) {
        float t = 0.f;
#pragma unroll
        for (int k = 0; k < 16; ++k) t += red[k][threadIdx.x];
        table_set(dtable, tdtype, (long)b * heads + h, t);
    }
}

template <typename T> constexpr int grad_vec() { return sizeof(T) == 2 ? 8 : 4; }
int grad_bands(int q_len) { return (q_len + GRAD_ROWS - 1) / GRAD_ROWS; }
int grad_blocks(int k_len, int vec) { return (k_len + GRAD_ROWS - 1 + 256 * vec - 1) / (256 * vec); }

template <typename T>
int bias_t(const void* table, int tdtype, const int32_t* map, int nb, int span, int heads, int q_len, int k_len, void* out, hipStream_t st) {
    constexpr int VEC = 16 / sizeof(T);
    const long groups = ((long)q_len * k_len + VEC - 1) / VEC + 1;         // a head's plane may begin and end inside a group
    const dim3 grid((unsigned)((groups + 256 * BIAS_ITER - 1) / (256 * BIAS_ITER)), heads);
    hipLaunchKernelGGL((rel_bias_kernel<T, VEC>), grid, dim3(256), 0, st, table, tdtype, map, nb, span, heads, q_len, k_len, reinterpret_cast<T*>(out));
    return (int)hipGetLastError();
}

template <typename T>
int grad_t(const void* dbias, const int32_t* map, int nb, int span, int batch, int heads, int q_len, int k_len, void* dtable, int tdtype, float* ws, hipStream_t st) {
    constexpr int VEC = grad_vec<T>();
    const int bands = grad_bands(q_len), blocks = grad_blocks(k_len, VEC), units = bands * blocks * 4;
    if (units > 0) hipLaunchKernelGGL((rel_bias_grad_kernel<T, VEC>), dim3(blocks, bands, heads), dim3(256), 0, st, reinterpret_cast<const T*>(dbias), map, nb, span,
                       batch, heads, q_len, k_len, units, ws);
    const int rc = (int)hipGetLastError();
    if (rc) return rc;
    hipLaunchKernelGGL(rel_bias_reduce_kernel, dim3((nb + 63) / 64, heads), dim3(1024), 0, st, ws, units, nb, heads, dtable, tdtype);
    return (int)hipGetLastError();
}

}  // namespace

int launch_rel_bias(int dtype, int tdtype, const void* table, const int32_t* map, int nb, int span, int heads, int q_len, int k_len, void* out, hipStream_t st) {
    return dtype == CV_DTYPE_F16 ? bias_t<half_t>(table, tdtype, map, nb, span, heads, q_len, k_len, out, st)
         : dtype == CV_DTYPE_BF16 ? bias_t<bhalf_t>(table, tdtype, map, nb, span, heads, q_len, k_len, out, st)
                                  : bias_t<float>(table, tdtype, map, nb, span, heads, q_len, k_len, out, st);
}
int64_t rel_bias_grad_ws(int nb, int heads, int q_len, int k_len) {
    return (int64_t)heads * grad_bands(q_len) * grad_blocks(k_len, 4) * 4 * nb * 4;     // the fp32 form has the most units
}
int launch_rel_bias_grad(int dtype, int tdtype, const void* dbias, const int32_t* map, int nb, int span, int batch, int heads, int q_len, int k_len, void* dtable,
                         float* ws, hipStream_t st) {
    return dtype == CV_DTYPE_F16 ? grad_t<half_t>(dbias, map, nb, span, batch, heads, q_len, k_len, dtable, tdtype, ws, st)
         : dtype == CV_DTYPE_BF16 ? grad_t<bhalf_t>(dbias, map, nb, span, batch, heads, q_len, k_len, dtable, tdtype, ws, st)
                                  : grad_t<float>(dbias, map, nb, span, batch, heads, q_len, k_len, dtable, tdtype, ws, st);
}

}  // namespace cva
