// Attention over the paged KV cache in 8 bits: one warp per query row, one
// lane per key for the scores, lanes across head_dim for the values.
#include "kv8.cuh"

namespace t2c {
namespace {

constexpr int kRowWarps = 4;

struct AttnArgs {
    KvPages pg;
    const __half *q;
    int64_t q_sb, q_st, q_sh;
    __half *out;
    int64_t o_sb, o_st, o_sh;
    float *lse;  // [B, NH, T]
    const int32_t *positions, *table;
    int64_t t_stride, max_len;
    int B, T, NH;
    float scale_log2;
};

// Number of keys query t of sequence b sees.
__device__ __forceinline__ int64_t visible(const int32_t *positions, int b, int t, int64_t max_len) {
    const int64_t n = static_cast<int64_t>(positions[b]) + t + 1;
    if (n > max_len) {
        report_device_error(T2C_EINVAL);
        return max_len;
    }
    return n < 0 ? 0 : n;
}

__device__ __forceinline__ float dot_row(const int8_t *row, const float *q, int D) {
    float acc = 0.0f;
    for (int i = 0; i < D; i += 16) {
        const uint4 c = *reinterpret_cast<const uint4 *>(row + i);
        const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc = fmaf(static_cast<float>(static_cast<int8_t>(w[j] >> (8 * e))), q[i + 4 * j + e], acc);
    }
    return acc;
}

template <int D>
__global__ void __launch_bounds__(32 * kRowWarps) attn8_row_kernel(AttnArgs a) {
    __shared__ float qs[kRowWarps][D];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t row = static_cast<int64_t>(blockIdx.x) * kRowWarps + warp;
    pdl_wait();
    pdl_trigger();
    if (row >= static_cast<int64_t>(a.B) * a.T * a.NH) return;
    const int h = static_cast<int>(row % a.NH), t = static_cast<int>(row / a.NH % a.T);
    const int b = static_cast<int>(row / a.NH / a.T);
    const int head = h / (a.NH / a.pg.n_kv);
    const __half *q = a.q + b * a.q_sb + t * a.q_st + h * a.q_sh;
    for (int i = lane; i < D; i += 32) qs[warp][i] = __half2float(q[i]);
    __syncwarp();
    const int64_t n = visible(a.positions, b, t, a.max_len);
    const int32_t *bt = a.table + b * a.t_stride;
    float m = -INFINITY, l = 0.0f, acc[D / 32] = {};
    for (int64_t base = 0; base < n; base += 32) {
        const int64_t key = base + lane;
        float x = -INFINITY, vs = 0.0f;
        int64_t off = 0;
        if (key < n) {
            int page = kv8_page(a.pg, bt, key);
            if (page < 0) page = 0;
            off = kv8_row_offset(a.pg, page, head, key);
            const int64_t so = kv8_scale_offset(a.pg, page, head, key);
            vs = __half2float(a.pg.vs[so]);
            x = dot_row(a.pg.k + off, qs[warp], D) * __half2float(a.pg.ks[so]) * a.scale_log2;
        }
        const float m_new = fmaxf(m, warp_max(x));
        const float corr = m == -INFINITY ? 0.0f : exp2f(m - m_new);
        const float p = key < n ? exp2f(x - m_new) : 0.0f;
        l = l * corr + warp_sum(p);
        m = m_new;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) acc[i] *= corr;
        const float pv = p * vs;
        const int count = static_cast<int>(n - base < 32 ? n - base : 32);
        for (int j = 0; j < count; ++j) {
            const float w = __shfl_sync(0xffffffffu, pv, j);
            const int8_t *v = a.pg.v + __shfl_sync(0xffffffffu, off, j);
#pragma unroll
            for (int i = 0; i < D / 32; ++i) acc[i] = fmaf(w, static_cast<float>(v[32 * i + lane]), acc[i]);
        }
    }
    __half *out = a.out + b * a.o_sb + t * a.o_st + h * a.o_sh;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) out[32 * i + lane] = __float2half(n > 0 ? acc[i] / l : 0.0f);
    if (a.lse && lane == 0)
        a.lse[(static_cast<int64_t>(b) * a.NH + h) * a.T + t] = n > 0 ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
}

// One warp per (sequence, KV head, 32 keys): a lane's key against every query that sees it.
template <int D>
__global__ void __launch_bounds__(32) attn8_weights_kernel(AttnArgs a, const float *lse, const float *w_in, float *w_out,
                                                           int64_t w_sb, int64_t w_sh) {
    __shared__ float qs[D];
    const int lane = threadIdx.x;
    const int head = blockIdx.y, b = blockIdx.z;
    pdl_wait();
    pdl_trigger();
    const int64_t first = a.positions[b];
    const int64_t n = visible(a.positions, b, a.T - 1, a.max_len);
    const int64_t key = static_cast<int64_t>(blockIdx.x) * 32 + lane;
    if (key - lane >= n) return;
    const int64_t at = key < n ? key : n - 1;
    int page = kv8_page(a.pg, a.table + b * a.t_stride, at);
    if (page < 0) page = 0;
    const int8_t *row = a.pg.k + kv8_row_offset(a.pg, page, head, at);
    const float s = __half2float(a.pg.ks[kv8_scale_offset(a.pg, page, head, at)]) * a.scale_log2;
    const int group = a.NH / a.pg.n_kv;
    float sum = 0.0f;
    for (int t = 0; t < a.T; ++t) {
        if (first + t < key - lane) continue;
        for (int g = 0; g < group; ++g) {
            const int h = head * group + g;
            __syncwarp();
            for (int i = lane; i < D; i += 32) qs[i] = __half2float(a.q[b * a.q_sb + t * a.q_st + h * a.q_sh + i]);
            __syncwarp();
            const float x = dot_row(row, qs, D) * s;
            if (key <= first + t)
                sum += exp2f(x - lse[(static_cast<int64_t>(b) * a.NH + h) * a.T + t] * 1.4426950408889634f);
        }
    }
    if (key >= n) return;
    const int64_t o = b * w_sb + head * w_sh + key;
    w_out[o] = sum + (w_in && key < first ? w_in[o] : 0.0f);
}

int check(const t2c_q8_pages *pages, const char *what, KvPages &pg, const int32_t *table, int64_t bt_stride,
          int64_t bt_width, const int32_t *positions, int64_t B, int64_t T, int64_t NH, int64_t &max_len) {
    int64_t capacity = 0;
    int rc = kv8_view(pages, what, pg);
    if (rc == T2C_OK) rc = kv8_table(pages, table, bt_stride, bt_width, what, capacity);
    if (rc != T2C_OK) return rc;
    if (!positions) return set_error(T2C_EINVAL, "%s: NULL positions", what);
    if (B <= 0 || T <= 0 || NH <= 0 || NH % pg.n_kv || B > 65535 || B * T * NH > INT32_MAX)
        return set_error(T2C_EINVAL, "%s: bad shape", what);
    if (max_len <= 0 || max_len > capacity) max_len = capacity;
    return T2C_OK;
}

int launch_weights(const AttnArgs &a, const float *lse, const float *weights, float *weights_out, int64_t w_sb,
                   int64_t w_sh, int64_t D, cudaStream_t s) {
    const dim3 grid(static_cast<unsigned>((a.max_len + 31) / 32), static_cast<unsigned>(a.pg.n_kv), static_cast<unsigned>(a.B));
    return kv8_launch("attn_key_weights_q8", D == 128 ? attn8_weights_kernel<128> : attn8_weights_kernel<64>, grid, dim3(32), 0,
                      1, s, a, lse, weights, weights_out, w_sb, w_sh);
}

int launch_rows(const AttnArgs &a, int64_t D, cudaStream_t s) {
    const int64_t rows = static_cast<int64_t>(a.B) * a.T * a.NH;
    return kv8_launch("attn_q8", D == 128 ? attn8_row_kernel<128> : attn8_row_kernel<64>,
                      dim3(static_cast<unsigned>((rows + kRowWarps - 1) / kRowWarps)), dim3(32 * kRowWarps), 0, 1, s, a);
}

bool strides_ok(const void *p, int64_t a, int64_t b, int64_t c) {
    return p && kv8_aligned(p, 16) && a % 8 == 0 && b % 8 == 0 && c % 8 == 0;
}

}  // namespace

cudaError_t status_attn8(unsigned int *bits, int clear, cudaStream_t s) { return read_tu_status(bits, clear, s); }

}  // namespace t2c

using namespace t2c;

extern "C" int64_t t2c_attn_decode_q8_workspace(const t2c_q8_pages *pages, int64_t bt_width, int64_t B, int64_t NH,
                                                int64_t max_len, int64_t splits, int with_weights) {
    (void)pages, (void)bt_width, (void)max_len, (void)splits;
    return with_weights ? B * NH : 0;
}

extern "C" int t2c_attn_decode_q8(const t2c_q8_pages *pages, const void *q, int64_t q_sb, int64_t q_sh, void *out,
                                  int64_t o_sb, int64_t o_sh, float *lse, const int32_t *positions,
                                  const int32_t *block_table, int64_t bt_stride, int64_t bt_width, int64_t B, int64_t NH,
                                  float scale, int64_t max_len, int64_t splits, const float *weights, float *weights_out,
                                  int64_t w_sb, int64_t w_sh, float *workspace, int64_t workspace_floats, void *stream) {
    AttnArgs a = {};
    int rc = check(pages, "attn_decode_q8", a.pg, block_table, bt_stride, bt_width, positions, B, 1, NH, max_len);
    if (rc != T2C_OK) return rc;
    if (!strides_ok(q, q_sb, q_sh, 0) || !strides_ok(out, o_sb, o_sh, 0))
        return set_error(T2C_EINVAL, "attn_decode_q8: q and out rows must be 16-byte aligned");
    if (splits < 0) return set_error(T2C_EINVAL, "attn_decode_q8: splits %lld", (long long)splits);
    const int64_t need = t2c_attn_decode_q8_workspace(pages, bt_width, B, NH, max_len, splits, weights_out != nullptr);
    if (need > 0 && (!workspace || workspace_floats < need))
        return set_error(T2C_ESCRATCH, "attn_decode_q8: workspace needs %lld floats", (long long)need);
    a.q = static_cast<const __half *>(q), a.q_sb = q_sb, a.q_sh = q_sh;
    a.out = static_cast<__half *>(out), a.o_sb = o_sb, a.o_sh = o_sh;
    a.lse = lse ? lse : (weights_out ? workspace : nullptr);
    a.positions = positions, a.table = block_table, a.t_stride = bt_stride, a.max_len = max_len;
    a.B = static_cast<int>(B), a.T = 1, a.NH = static_cast<int>(NH);
    a.scale_log2 = scale * 1.4426950408889634f;
    rc = launch_rows(a, pages->head_dim, as_stream(stream));
    if (rc == T2C_OK && weights_out)
        rc = launch_weights(a, a.lse, weights, weights_out, w_sb, w_sh, pages->head_dim, as_stream(stream));
    return rc;
}

extern "C" int64_t t2c_attn_prefill_q8_workspace(const t2c_q8_pages *pages, int64_t bt_width, int64_t B, int64_t T,
                                                 int64_t NH, int64_t max_len, int64_t splits) {
    (void)pages, (void)bt_width, (void)B, (void)T, (void)NH, (void)max_len, (void)splits;
    return 0;
}

extern "C" int t2c_attn_prefill_q8(const t2c_q8_pages *pages, const void *q, int64_t q_sb, int64_t q_st, int64_t q_sh,
                                   void *out, int64_t o_sb, int64_t o_st, int64_t o_sh, float *lse,
                                   const int32_t *positions, const int32_t *block_table, int64_t bt_stride,
                                   int64_t bt_width, int64_t B, int64_t T, int64_t NH, float scale, int64_t max_len,
                                   int64_t splits, float *workspace, int64_t workspace_floats, void *stream) {
    AttnArgs a = {};
    int rc = check(pages, "attn_prefill_q8", a.pg, block_table, bt_stride, bt_width, positions, B, T, NH, max_len);
    if (rc != T2C_OK) return rc;
    if (!strides_ok(q, q_sb, q_st, q_sh) || !strides_ok(out, o_sb, o_st, o_sh))
        return set_error(T2C_EINVAL, "attn_prefill_q8: q and out rows must be 16-byte aligned");
    if (splits < 0) return set_error(T2C_EINVAL, "attn_prefill_q8: splits %lld", (long long)splits);
    const int64_t need = t2c_attn_prefill_q8_workspace(pages, bt_width, B, T, NH, max_len, splits);
    if (need > 0 && (!workspace || workspace_floats < need))
        return set_error(T2C_ESCRATCH, "attn_prefill_q8: workspace needs %lld floats", (long long)need);
    a.q = static_cast<const __half *>(q), a.q_sb = q_sb, a.q_st = q_st, a.q_sh = q_sh;
    a.out = static_cast<__half *>(out), a.o_sb = o_sb, a.o_st = o_st, a.o_sh = o_sh;
    a.lse = lse;
    a.positions = positions, a.table = block_table, a.t_stride = bt_stride, a.max_len = max_len;
    a.B = static_cast<int>(B), a.T = static_cast<int>(T), a.NH = static_cast<int>(NH);
    a.scale_log2 = scale * 1.4426950408889634f;
    return launch_rows(a, pages->head_dim, as_stream(stream));
}

extern "C" int t2c_attn_key_weights_q8(const t2c_q8_pages *pages, const void *q, int64_t q_sb, int64_t q_st,
                                       int64_t q_sh, const float *lse, const int32_t *positions,
                                       const int32_t *block_table, int64_t bt_stride, int64_t bt_width, int64_t B,
                                       int64_t T, int64_t NH, float scale, int64_t max_len, const float *weights,
                                       float *weights_out, int64_t w_sb, int64_t w_sh, void *stream) {
    AttnArgs a = {};
    int rc = check(pages, "attn_key_weights_q8", a.pg, block_table, bt_stride, bt_width, positions, B, T, NH, max_len);
    if (rc != T2C_OK) return rc;
    if (!strides_ok(q, q_sb, q_st, q_sh)) return set_error(T2C_EINVAL, "attn_key_weights_q8: q rows must be 16-byte aligned");
    if (!lse || !weights_out) return set_error(T2C_EINVAL, "attn_key_weights_q8: NULL pointer");
    a.q = static_cast<const __half *>(q), a.q_sb = q_sb, a.q_st = q_st, a.q_sh = q_sh;
    a.positions = positions, a.table = block_table, a.t_stride = bt_stride, a.max_len = max_len;
    a.B = static_cast<int>(B), a.T = static_cast<int>(T), a.NH = static_cast<int>(NH);
    a.scale_log2 = scale * 1.4426950408889634f;
    return launch_weights(a, lse, weights, weights_out, w_sb, w_sh, pages->head_dim, as_stream(stream));
}
