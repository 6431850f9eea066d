// C entries of the sequence operators: every argument is checked here, so that the kernels never see a shape they do not cover.
#include <math.h>

#include "seqops.h"

using namespace cva;

#define REFUSE(code, ...) do { cva_set_error(__VA_ARGS__); return code; } while (0)

namespace {

constexpr int64_t LAUNCH_GROUPS = 1 << 24;       // workgroups of 256 threads
constexpr int64_t MOST_ROWS = 0x7fffffff;        // offsets are int32

bool dtype_ok(int d) { return d == CV_DTYPE_F16 || d == CV_DTYPE_BF16 || d == CV_DTYPE_F32; }
int size_of(int d) { return d == CV_DTYPE_F32 ? 4 : 2; }
bool aligned(const void* p, size_t n) { return ((uintptr_t)p) % n == 0; }
hipStream_t stream_of(void* s) { return reinterpret_cast<hipStream_t>(s); }
int launched(int rc, const char* what) {
    if (rc) { cva_set_error("%s: launch failed (%s)", what, hipGetErrorString((hipError_t)rc)); return CV_ERR_HIP; }
    return CV_OK;
}

// ---- bucket map: is (span / e)^k <= (d / e)^n, i.e. span^k e^(n - k) <= d^n ?  Whole numbers of up to 128 words.
struct Big { uint32_t w[160]; int n; };
void big_mul(Big& b, uint32_t f) {
    uint64_t carry = 0;
    for (int i = 0; i < b.n; ++i) { carry += (uint64_t)b.w[i] * f; b.w[i] = (uint32_t)carry; carry >>= 32; }
    if (carry) b.w[b.n++] = (uint32_t)carry;
}
bool reaches(int span, int e, int d, int k, int n) {
    Big l{}, r{};
    l.w[0] = r.w[0] = 1; l.n = r.n = 1;
    for (int i = 0; i < n; ++i) { big_mul(l, (uint32_t)(i < k ? span : e)); big_mul(r, (uint32_t)d); }
    if (l.n != r.n) return l.n < r.n;
    for (int i = l.n - 1; i >= 0; --i)
        if (l.w[i] != r.w[i]) return l.w[i] < r.w[i];
    return true;
}
int side_bucket(int d, int n, int span) {
    const int e = n / 2, steps = n - e;
    if (d < e) return d;
    int k = (int)(steps * log((double)d / e) / log((double)span / e));        // within one of the answer; whole numbers decide
    if (k < 0) k = 0;
    if (k > steps - 1) k = steps - 1;
    while (k + 1 < steps && reaches(span, e, d, k + 1, steps)) ++k;
    while (k > 0 && !reaches(span, e, d, k, steps)) --k;
    return e + k;
}

int check_map(const char* fn, int dtype, int tdtype, const int32_t* map, int nb, int span) {
    if (nb < 1 || nb > 256) REFUSE(CV_ERR_INVALID, "%s: num_buckets must be 1 .. 256 (got %d)", fn, nb);
    if (span < 0 || span > 65536) REFUSE(CV_ERR_INVALID, "%s: span must be 0 .. 65536 (got %d)", fn, span);
    if (!map) REFUSE(CV_ERR_INVALID, "%s: the bucket map is missing", fn);
    if (tdtype != CV_DTYPE_F32 && tdtype != dtype) REFUSE(CV_ERR_INVALID, "%s: the table must be f32 or of the call's dtype", fn);
    return CV_OK;
}
int check_plane(const char* fn, int dtype, int heads, int q_len, int k_len) {
    if (!dtype_ok(dtype)) REFUSE(CV_ERR_INVALID, "%s: dtype must be f16, bf16 or f32", fn);
    if (heads < 1 || heads > 65535 || q_len < 0 || k_len < 0 || q_len > (1 << 22) || k_len > (1 << 22))
        REFUSE(CV_ERR_INVALID, "%s: bad sizes (heads %d, q_len %d, k_len %d)", fn, heads, q_len, k_len);
    return CV_OK;
}

// everything that the plans and the workspace sizes rely on
int check_attn_shape(const char* fn, const cv_rel_attn* a, bool grad) {
    if (!a) REFUSE(CV_ERR_INVALID, "%s: null argument", fn);
    if (!dtype_ok(a->dtype)) REFUSE(CV_ERR_INVALID, "%s: dtype must be f16, bf16 or f32", fn);
    if (a->n_seq < 0 || a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads != 0 || a->heads > 65536)
        REFUSE(CV_ERR_INVALID, "%s: %d query heads over %d key heads", fn, a->heads, a->kv_heads);
    const int G = a->heads / a->kv_heads;
    if (G > 32) REFUSE(CV_ERR_UNSUPPORTED, "%s: at most 32 query heads share a key head (got %d)", fn, G);
    if (a->head_dim < 8 || a->head_dim > 128 || a->head_dim % 8) REFUSE(CV_ERR_UNSUPPORTED, "%s: head_dim must be a multiple of 8 up to 128 (got %d)", fn, a->head_dim);
    if (a->max_q < 0 || a->max_k < 0 || (int64_t)a->max_q * G > (1 << 28) || a->max_k > (1 << 28)) REFUSE(CV_ERR_INVALID, "%s: bad lengths (max_q %d, max_k %d)", fn, a->max_q, a->max_k);
    if ((a->q_off && a->rows_q < 0) || (a->k_off && a->rows_k < 0)) REFUSE(CV_ERR_INVALID, "%s: negative number of rows", fn);
    if ((a->q_off && a->rows_q > MOST_ROWS) || (a->k_off && a->rows_k > MOST_ROWS)) REFUSE(CV_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 packed rows", fn);
    if ((a->table || a->dtable) && (a->num_buckets < 1 || a->num_buckets > 256)) REFUSE(CV_ERR_INVALID, "%s: num_buckets must be 1 .. 256 (got %d)", fn, a->num_buckets);
    if ((a->table || a->dtable) && (a->span < 0 || a->span > 65536)) REFUSE(CV_ERR_INVALID, "%s: span must be 0 .. 65536 (got %d)", fn, a->span);
    // a launch has less than 2^32 threads, 256 a workgroup
    const int64_t pairs = (int64_t)a->kv_heads * a->n_seq;
    if (pairs >= LAUNCH_GROUPS || (rel_attention_tiles(*a, grad) * ((pairs + 7) & ~7LL)) >= LAUNCH_GROUPS) REFUSE(CV_ERR_UNSUPPORTED, "%s: too many tiles for one launch", fn);
    return CV_OK;
}

int check_attn(const cv_rel_attn* a, bool grad) {
    const char* fn = grad ? "cv_op_rel_attention_grad" : "cv_op_rel_attention";
    if (const int rc = check_attn_shape(fn, a, grad)) return rc;
    const int G = a->heads / a->kv_heads;
    if (!(a->scale >= 1e-6f && a->scale <= 1e6f)) REFUSE(CV_ERR_INVALID, "%s: scale must lie in 1e-6 .. 1e6", fn);
    if (a->table) {
        const int rc = check_map(fn, a->dtype, a->table_dtype, a->map, a->num_buckets, a->span);
        if (rc) return rc;
    }
    if (a->dtable && !a->table) REFUSE(CV_ERR_INVALID, "%s: dtable without a table", fn);
    const int64_t e = 16 / size_of(a->dtype);
    const int64_t strides[] = {a->q_seq, a->q_row, a->q_head, a->k_seq, a->k_row, a->k_head, a->v_seq, a->v_row, a->v_head, a->o_seq, a->o_row, a->o_head};
    for (int64_t s : strides)
        if (s % e) REFUSE(CV_ERR_INVALID, "%s: strides must be multiples of %d elements", fn, (int)e);
    if (grad && (a->do_seq % e || a->do_row % e || a->do_head % e)) REFUSE(CV_ERR_INVALID, "%s: strides must be multiples of %d elements", fn, (int)e);
    // inside a tile offsets are 32-bit: 128 positions of a head group, 64 keys
    const int64_t es = size_of(a->dtype);
    const int64_t steps[] = {a->q_seq, a->q_row, a->q_head, a->k_seq, a->k_row, a->k_head, a->v_seq, a->v_row, a->v_head, a->o_seq, a->o_row, a->o_head,
                             a->do_seq, a->do_row, a->do_head};
    for (int64_t s : steps)
        if (s < 0) REFUSE(CV_ERR_INVALID, "%s: negative stride", fn);
    const int64_t row_most = (int64_t)1 << 24;
    if (a->q_row * es > row_most || a->k_row * es > row_most || a->v_row * es > row_most || a->do_row * es > row_most || (G - 1) * a->q_head * es > ((int64_t)1 << 30) - 256 ||
        (G - 1) * a->do_head * es > ((int64_t)1 << 30) - 256)
        REFUSE(CV_ERR_UNSUPPORTED, "%s: row strides beyond 16 MiB or heads of a group beyond 1 GiB apart", fn);
    const bool qs = a->n_seq > 0 && a->max_q > 0 && (!a->q_off || a->rows_q > 0), ks = a->n_seq > 0 && a->max_k > 0 && (!a->k_off || a->rows_k > 0);
    if ((qs && (!a->q || !a->out)) || (ks && (!a->k || !a->v))) REFUSE(CV_ERR_INVALID, "%s: null argument", fn);
    const void* ptrs[] = {a->q, a->k, a->v, a->out, a->out_lo, a->ws};
    for (const void* p : ptrs)
        if (!aligned(p, 16)) REFUSE(CV_ERR_INVALID, "%s: pointers must be 16-byte aligned", fn);
    if (grad) {
        if ((qs && (!a->dout || !a->lse || !a->dq)) || (ks && (!a->dk || !a->dv))) REFUSE(CV_ERR_INVALID, "%s: null argument", fn);
        const void* more[] = {a->dout, a->dq, a->dk, a->dv};
        for (const void* p : more)
            if (!aligned(p, 16)) REFUSE(CV_ERR_INVALID, "%s: pointers must be 16-byte aligned", fn);
    }
    return CV_OK;
}

int check_norm(const cv_block_norm* a, bool grad) {
    const char* fn = grad ? "cv_op_block_norm_grad" : "cv_op_block_norm";
    if (!a) REFUSE(CV_ERR_INVALID, "%s: null argument", fn);
    if (!dtype_ok(a->dtype)) REFUSE(CV_ERR_INVALID, "%s: dtype must be f16, bf16 or f32", fn);
    if (a->kind != 0 && a->kind != 1) REFUSE(CV_ERR_INVALID, "%s: kind must be 0 (LayerNorm) or 1 (RMSNorm)", fn);
    if (a->M < 0 || a->M >= LAUNCH_GROUPS || a->C < 1 || a->C > 8192) REFUSE(CV_ERR_UNSUPPORTED, "%s: 0 <= M < 2^24 and 1 <= C <= 8192 required (got %d, %d)", fn, a->M, a->C);
    if (!(a->eps >= 0.f) || !isfinite(a->eps) || !isfinite(a->alpha)) REFUSE(CV_ERR_INVALID, "%s: eps must be >= 0, alpha finite", fn);
    if (a->gate && a->rows_per_gate < 1) REFUSE(CV_ERR_INVALID, "%s: rows_per_gate must be positive", fn);
    if (a->M > 0 && (!a->y || (!grad && (!a->x || !a->x_out)))) REFUSE(CV_ERR_INVALID, "%s: null argument", fn);
    const bool rows = a->M > 1;
    if (rows && (a->y_row < a->C || (!grad && (a->x_row < a->C || a->xo_row < a->C || (a->z && a->z_row < a->C))) ||
                 (grad && ((a->dx_out && a->dxo_row < a->C) || (a->dz && (a->dz_row < a->C || a->xo_row < a->C))))))
        REFUSE(CV_ERR_INVALID, "%s: a row stride is shorter than a row", fn);
    const void* f32s[] = {a->x, a->post_w, a->post_b, a->gate, a->pre_w, a->pre_b, a->x_out, a->dx_out, a->dx};
    for (const void* p : f32s)
        if (!aligned(p, 4)) REFUSE(CV_ERR_INVALID, "%s: misaligned pointer", fn);
    const void* ts[] = {a->y, a->z, a->dz, a->dy};
    for (const void* p : ts)
        if (!aligned(p, size_of(a->dtype))) REFUSE(CV_ERR_INVALID, "%s: misaligned pointer", fn);
    if (!aligned(a->stats, 16) || !aligned(a->ws, 16)) REFUSE(CV_ERR_INVALID, "%s: stats and ws must be 16-byte aligned", fn);
    if (grad && a->M > 0) {
        if (!a->stats || (a->dz && !a->x_out)) REFUSE(CV_ERR_INVALID, "%s: stats (and x_out with dz) of the forward are missing", fn);
    }
    return CV_OK;
}

}  // namespace

extern "C" int cv_rel_buckets_host(int num_buckets, int span, int bidirectional, int32_t* map) {
    const int side = bidirectional ? num_buckets / 2 : num_buckets;
    if (!map) REFUSE(CV_ERR_INVALID, "cv_rel_buckets_host: null argument");
    if (num_buckets < 2 || num_buckets > 256 || (bidirectional && (num_buckets % 2 || side < 2)))
        REFUSE(CV_ERR_INVALID, "cv_rel_buckets_host: num_buckets must be 2 .. 256, even and at least 4 for both directions (got %d)", num_buckets);
    if (span <= side / 2 || span > 65536) REFUSE(CV_ERR_INVALID, "cv_rel_buckets_host: span must lie in %d .. 65536 (got %d)", side / 2 + 1, span);
    for (int d = 0; d <= span; ++d) {
        const int b = side_bucket(d, side, span);
        map[span - d] = b;
        if (d) map[span + d] = bidirectional ? side + b : 0;
    }
    return CV_OK;
}

extern "C" int cv_op_rel_bias(int dtype, int table_dtype, const void* table, const int32_t* map, int num_buckets, int span, int heads, int q_len, int k_len, void* out,
                              void* stream) {
    int rc = check_plane("cv_op_rel_bias", dtype, heads, q_len, k_len);
    if (rc || (rc = check_map("cv_op_rel_bias", dtype, table_dtype, map, num_buckets, span))) return rc;
    if (q_len == 0 || k_len == 0) return CV_OK;
    if (!table || !out) REFUSE(CV_ERR_INVALID, "cv_op_rel_bias: null argument");
    if (!aligned(out, 16)) REFUSE(CV_ERR_INVALID, "cv_op_rel_bias: out must be 16-byte aligned");
    return launched(launch_rel_bias(dtype, table_dtype, table, map, num_buckets, span, heads, q_len, k_len, out, stream_of(stream)), "cv_op_rel_bias");
}
extern "C" int64_t cv_op_rel_bias_grad_ws(int num_buckets, int heads, int q_len, int k_len) {
    if (check_plane("cv_op_rel_bias_grad_ws", CV_DTYPE_F32, heads, q_len, k_len) || num_buckets < 1 || num_buckets > 256) return -1;
    return rel_bias_grad_ws(num_buckets, heads, q_len, k_len);
}
extern "C" int cv_op_rel_bias_grad(int dtype, int table_dtype, const void* dbias, const int32_t* map, int num_buckets, int span, int batch, int heads, int q_len, int k_len,
                                   void* dtable, void* ws, int64_t ws_bytes, void* stream) {
    int rc = check_plane("cv_op_rel_bias_grad", dtype, heads, q_len, k_len);
    if (rc || (rc = check_map("cv_op_rel_bias_grad", dtype, table_dtype, map, num_buckets, span))) return rc;
    if (batch < 0 || !dtable) REFUSE(CV_ERR_INVALID, "cv_op_rel_bias_grad: null argument");
    if (batch > 0 && q_len > 0 && k_len > 0 && !dbias) REFUSE(CV_ERR_INVALID, "cv_op_rel_bias_grad: null argument");
    if (!aligned(dbias, size_of(dtype))) REFUSE(CV_ERR_INVALID, "cv_op_rel_bias_grad: misaligned pointer");
    if (ws_bytes < rel_bias_grad_ws(num_buckets, heads, q_len, k_len) || (q_len > 0 && !ws) || !aligned(ws, 16))
        REFUSE(CV_ERR_INVALID, "cv_op_rel_bias_grad: the workspace is too small or misaligned");
    if (k_len == 0 || q_len == 0) batch = 0;
    return launched(launch_rel_bias_grad(dtype, table_dtype, dbias, map, num_buckets, span, batch, heads, q_len, k_len, dtable, reinterpret_cast<float*>(ws),
                                         stream_of(stream)), "cv_op_rel_bias_grad");
}

extern "C" int64_t cv_op_rel_attention_ws(const cv_rel_attn* a, int grad) {
    if (const int rc = check_attn_shape("cv_op_rel_attention_ws", a, grad != 0)) return -rc;
    return grad ? rel_attention_bwd_ws(*a) : rel_attention_fwd_ws(*a);
}
extern "C" int cv_op_rel_attention(const cv_rel_attn* a, void* stream) {
    const int rc = check_attn(a, false);
    if (rc) return rc;
    const int64_t need = rel_attention_fwd_ws(*a);
    if (need && (!a->ws || a->ws_bytes < need)) REFUSE(CV_ERR_INVALID, "cv_op_rel_attention: the workspace is too small (%lld bytes needed)", (long long)need);
    return launched(launch_rel_attention(*a, stream_of(stream)), "cv_op_rel_attention");
}
extern "C" int cv_op_rel_attention_grad(const cv_rel_attn* a, void* stream) {
    const int rc = check_attn(a, true);
    if (rc) return rc;
    const int64_t need = rel_attention_bwd_ws(*a);
    if (!a->ws || a->ws_bytes < need) REFUSE(CV_ERR_INVALID, "cv_op_rel_attention_grad: the workspace is too small (%lld bytes needed)", (long long)need);
    return launched(launch_rel_attention_grad(*a, stream_of(stream)), "cv_op_rel_attention_grad");
}

extern "C" int cv_op_block_norm(const cv_block_norm* a, void* stream) {
    const int rc = check_norm(a, false);
    if (rc || a->M == 0) return rc;
    return launched(launch_block_norm(*a, stream_of(stream)), "cv_op_block_norm");
}
extern "C" int64_t cv_op_block_norm_grad_ws(const cv_block_norm* a) {
    return check_norm(a, true) ? -1 : block_norm_grad_ws(*a);
}
extern "C" int cv_op_block_norm_grad(const cv_block_norm* a, void* stream) {
    const int rc = check_norm(a, true);
    if (rc) return rc;
    const int64_t need = block_norm_grad_ws(*a);
    if (need && (!a->ws || a->ws_bytes < need)) REFUSE(CV_ERR_INVALID, "cv_op_block_norm_grad: the workspace is too small (%lld bytes needed)", (long long)need);
    return launched(launch_block_norm_grad(*a, stream_of(stream)), "cv_op_block_norm_grad");
}
static_assert(sizeof(cv_rel_attn) == 328 && sizeof(cv_block_norm) == 248, "the ctypes binding mirrors these structs field by field");
