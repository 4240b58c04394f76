// Attention over the paged KV cache in 8 bits: one warp per query row, one
// lane per key for the scores, lanes across head_dim for the values.
#include <cooperative_groups.h>

#include "kv8.cuh"

namespace cg = cooperative_groups;

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

// ------------------------------------------------------------------ one token per sequence
// A warp walks its share of a sequence's keys in steps of 16.  Codes arrive by 16-byte cp.async in a ring of
// kDStages steps that only this warp reads (no CTA barrier in the loop); a step's 16 keys lie in one block, so one K
// and one V scale serve it.  Both products run on mma.m16n8k16 with the up to 8 heads of a group as the n side, so
// that a cached byte is expanded once for all of them:
//   S^T [16 keys x 8 heads] = K Q^T,   O^T [16 dims x 8 heads] += V^T P^T.
// Codes become fp16 exactly.  The scales stay in fp32: x = s * (k scale * softmax scale * log2 e), and the V scale
// joins the exponent, P = 2^(x + log2 vs - m), so that P q_v needs no scaled V; the softmax sum takes P / vs.  m is a
// running reference per head, moved (and O, l rescaled) only when some exponent passes 14: P stays in fp16's range,
// and its one rounding to fp16, shared with every attention kernel here, is the only one before the output.
// What bounds it: HBM.
constexpr int kDWarps = 4;
constexpr int kDStages = 3;
constexpr int kDThreads = 32 * kDWarps;
constexpr float kRefStart = -1e30f;  // below any finite score: the first step moves it
constexpr float kRefTop = 14.0f;     // P <= 2^14
constexpr float kRefDrop = 8.0f;     // a moved reference leaves the largest P at 2^8

template <int D>
struct DecodeShape {
    static constexpr int kChunks = D / 16;                     // 16-byte chunks of a row
    static constexpr int kStep = 16 * D;                       // bytes of K (or V) per step
    static constexpr int kRing = kDWarps * kDStages * 2 * kStep;
    // 16-byte slot of chunk c of row r: the fragment reads below touch each bank once per 8 lanes
    static __device__ __forceinline__ uint32_t slot(int r, int c) {
        if constexpr (D == 128) {
            return static_cast<uint32_t>(r * 8 + (c ^ (r & 7)));
        } else {
            const int j = r >> 1;
            return static_cast<uint32_t>(j * 8 + ((c & 1) | (((c >> 1) ^ ((j >> 1) & 1)) << 1) | (((r ^ j) & 1) << 2)));
        }
    }
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}

__device__ __forceinline__ void mma16816(float c[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}

__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }

// codes 0, 2 and 1, 3 of a word as two half2
__device__ __forceinline__ void unpack_word(uint32_t w, uint32_t &even, uint32_t &odd) {
    __half2 e, o;
    kv8_unpack(w, e, o);
    even = half2_bits(e);
    odd = half2_bits(o);
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct DecodeArgs {
    AttnArgs a;
    int splits, head_chunks;      // CTAs per (sequence, KV head); chunks of 8 heads of a group
    float *parts;                 // [B][n_kv * head_chunks][splits][8][D + 2]: O, m, l
    float *scores;                // [B][n_kv][s_len][group] x in log2 units, where the weights are wanted
    int64_t s_len;
    const float *w_in;
    float *w_out;
    int64_t w_sb, w_sh;
    bool join;                    // a second kernel joins the splits
};

// The keys that CTA `s` of `splits` takes of n: multiples of 16, at least 64 a CTA.
__device__ __forceinline__ void split_range(int64_t n, int splits, int s, int64_t &k0, int64_t &k1) {
    int64_t chunk = (n + splits - 1) / splits;
    chunk = chunk < 64 ? 64 : (chunk + 15) & ~int64_t(15);
    k0 = s * chunk < n ? s * chunk : n;
    k1 = k0 + chunk < n ? k0 + chunk : n;
}

__device__ __forceinline__ float key_weight(const float *x, const float *lse2, int group) {
    float sum = 0.0f;
    if ((group & 3) == 0) {  // rows of scores are 16-byte aligned
        for (int g = 0; g < group; g += 4) {
            const float4 v = *reinterpret_cast<const float4 *>(x + g);
            sum += exp2_approx(v.x - lse2[g]) + exp2_approx(v.y - lse2[g + 1]) + exp2_approx(v.z - lse2[g + 2]) +
                   exp2_approx(v.w - lse2[g + 3]);
        }
        return sum;
    }
    for (int g = 0; g < group; ++g) sum += exp2_approx(x[g] - lse2[g]);
    return sum;
}

template <int D>
__global__ void __launch_bounds__(kDThreads, 4) attn8_decode_kernel(DecodeArgs p) {
    using Shape = DecodeShape<D>;
    constexpr int kWords = D / 16;  // K: 32-bit words per lane and row = k steps; V: m tiles
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float st_m[kDWarps][8], st_l[kDWarps][8], cta_m[8], cta_l[8], lse2[8];
    const AttnArgs &a = p.a;
    cg::cluster_group cluster = cg::this_cluster();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x;
    const int head = blockIdx.y / p.head_chunks, chunk = blockIdx.y % p.head_chunks;
    const int b = blockIdx.z;
    const int group = a.NH / a.pg.n_kv, heads = min(8, group - 8 * chunk), h0 = head * group + 8 * chunk;
    pdl_wait();
    pdl_trigger();
    const int64_t n = visible(a.positions, b, 0, a.max_len);
    int64_t k0, k1;
    split_range(n, p.splits, split, k0, k1);
    const int32_t *bt = a.table + b * a.t_stride;
    const int steps = static_cast<int>((k1 - k0 + 15) >> 4);            // of the CTA
    const int mine = steps > warp ? (steps - warp + kDWarps - 1) / kDWarps : 0;  // of this warp: warp, warp + 4, ..

    // ---- the lane's step of a window of 32: page and scales, looked up a window ahead of their use
    int page = 0;
    float kf = 0.0f, lv = 0.0f, iv = 0.0f;
    const auto step_key = [&](int i) { return k0 + 16 * (warp + static_cast<int64_t>(kDWarps) * i); };
    const auto look_up_page = [&](int window) {
        const int i = window * 32 + lane;
        if (i < mine) page = max(kv8_page(a.pg, bt, step_key(i)), 0);
    };
    const auto look_up_scales = [&](int window) {
        const int i = window * 32 + lane;
        if (i >= mine) return;
        const int64_t so = kv8_scale_offset(a.pg, page, head, step_key(i));
        kf = __half2float(a.pg.ks[so]) * a.scale_log2;
        const float vs = __half2float(a.pg.vs[so]);
        // a block of scale 0 has values 0: any exponent adds nothing to O, the least scale's moves no reference
        lv = vs == 0.0f ? -24.0f : log2f(vs);
        iv = vs == 0.0f ? 16777216.0f : 1.0f / vs;
    };
    look_up_page(0);

    // ---- Q^T fragments: k step i, lane (g, t): head g, dims D/4 t + 4 i + {0, 2} and {1, 3}
    uint32_t qf[kWords][2];
    {
        const uint32_t *q = reinterpret_cast<const uint32_t *>(a.q + b * a.q_sb + (h0 + min(g, heads - 1)) * a.q_sh) + D / 8 * t;
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            const uint32_t lo = g < heads ? q[2 * i] : 0u, hi = g < heads ? q[2 * i + 1] : 0u;
            qf[i][0] = __byte_perm(lo, hi, 0x5410);
            qf[i][1] = __byte_perm(lo, hi, 0x7632);
        }
    }

    const uint32_t ring = smem_u32(smem) + warp * (kDStages * 2 * Shape::kStep);
    const int64_t row_in_page_mask = (1 << a.pg.page_log2) - 1;
    const int my_row = lane / Shape::kChunks, my_chunk = lane % Shape::kChunks;
    constexpr int kRowsPerPass = 32 / Shape::kChunks;
    const auto load = [&](int i, int from) {  // step i of this warp, whose page lane `from` knows
        if (i < mine) {
            const int64_t key = step_key(i);
            const int pg = __shfl_sync(0xffffffffu, page, from);
            const int64_t off = pg * a.pg.page_stride + head * a.pg.head_stride +
                                ((key & row_in_page_mask) + my_row) * a.pg.row_stride + 16 * my_chunk;
            const uint32_t st = ring + (i % kDStages) * 2 * Shape::kStep;
#pragma unroll
            for (int r = 0; r < 16 / kRowsPerPass; ++r) {
                const uint32_t dst = st + 16 * Shape::slot(my_row + r * kRowsPerPass, my_chunk);
                cp_async16(dst, a.pg.k + off + r * kRowsPerPass * a.pg.row_stride);
                cp_async16(dst + Shape::kStep, a.pg.v + off + r * kRowsPerPass * a.pg.row_stride);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };

    float o[kWords][4] = {};
    float m[2] = {kRefStart, kRefStart}, l[2] = {0.0f, 0.0f};
    float *xs = p.scores + ((static_cast<int64_t>(b) * a.pg.n_kv + head) * p.s_len) * group + 8 * chunk;
#pragma unroll
    for (int i = 0; i < kDStages - 1; ++i) load(i, i);
    look_up_scales(0);  // behind the first copies: their latencies overlap
    int next_page_lane = kDStages - 1;
    float cur_kf = kf, cur_lv = lv, cur_iv = iv;  // of the window being computed; kf, lv, iv: of the window being loaded
    for (int i = 0; i < mine; ++i) {
        if (next_page_lane == 32) {  // every page of the window has been used: look the next one up
            cur_kf = kf, cur_lv = lv, cur_iv = iv;
            look_up_page((i + kDStages - 1) / 32);
            look_up_scales((i + kDStages - 1) / 32);
            next_page_lane = 0;
        }
        load(i + kDStages - 1, next_page_lane++);
        asm volatile("cp.async.wait_group %0;" ::"n"(kDStages - 1) : "memory");
        __syncwarp();
        const bool same_window = (i + kDStages - 1) / 32 == i / 32;
        const float kf_i = __shfl_sync(0xffffffffu, same_window ? kf : cur_kf, i & 31);
        const float lv_i = __shfl_sync(0xffffffffu, same_window ? lv : cur_lv, i & 31);
        const float iv_i = __shfl_sync(0xffffffffu, same_window ? iv : cur_iv, i & 31);
        const uint32_t ks = ring + (i % kDStages) * 2 * Shape::kStep, vs = ks + Shape::kStep;
        const int64_t key = step_key(i);
        // S^T: rows g, g + 8 of K, the lane's D / 4 dims
        float s[4] = {};
#pragma unroll
        for (int c = 0; c < kWords / 4; ++c) {
            const uint4 lo = lds128(ks + 16 * Shape::slot(g, kWords / 4 * t + c));
            const uint4 hi = lds128(ks + 16 * Shape::slot(g + 8, kWords / 4 * t + c));
            const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                uint32_t a0, a1, a2, a3;
                unpack_word(wl[j], a0, a2);
                unpack_word(wh[j], a1, a3);
                mma16816(s, a0, a1, a2, a3, qf[4 * c + j][0], qf[4 * c + j][1]);
            }
        }
        // s[0], s[1]: key g, heads 2t, 2t + 1; s[2], s[3]: key g + 8
        const bool in0 = key + g < k1, in1 = key + g + 8 < k1;
        if (p.w_out) {
            float *x0 = xs + (key + g) * group + 2 * t, *x1 = x0 + 8 * group;
            if (in0 && 2 * t < heads) x0[0] = s[0] * kf_i;
            if (in0 && 2 * t + 1 < heads) x0[1] = s[1] * kf_i;
            if (in1 && 2 * t < heads) x1[0] = s[2] * kf_i;
            if (in1 && 2 * t + 1 < heads) x1[1] = s[3] * kf_i;
        }
        float y[4];
        y[0] = in0 ? fmaf(s[0], kf_i, lv_i - m[0]) : -INFINITY;
        y[1] = in0 ? fmaf(s[1], kf_i, lv_i - m[1]) : -INFINITY;
        y[2] = in1 ? fmaf(s[2], kf_i, lv_i - m[0]) : -INFINITY;
        y[3] = in1 ? fmaf(s[3], kf_i, lv_i - m[1]) : -INFINITY;
        if (__any_sync(0xffffffffu, fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])) > kRefTop)) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float top = fmaxf(in0 ? fmaf(s[e], kf_i, lv_i) : -INFINITY, in1 ? fmaf(s[2 + e], kf_i, lv_i) : -INFINITY);
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                const float ref = top - m[e] > kRefTop ? top - kRefDrop : m[e];
                const float corr = exp2_approx(m[e] - ref);
                l[e] *= corr;
#pragma unroll
                for (int w = 0; w < kWords; ++w) {
                    o[w][e] *= corr;
                    o[w][2 + e] *= corr;
                }
                m[e] = ref;
                y[e] = in0 ? fmaf(s[e], kf_i, lv_i - ref) : -INFINITY;
                y[2 + e] = in1 ? fmaf(s[2 + e], kf_i, lv_i - ref) : -INFINITY;
            }
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = exp2_approx(y[e]);
        l[0] = fmaf(y[0] + y[2], iv_i, l[0]);
        l[1] = fmaf(y[1] + y[3], iv_i, l[1]);
        const uint32_t b0 = transpose8x8(half2_bits(__floats2half2_rn(y[0], y[1])));
        const uint32_t b1 = transpose8x8(half2_bits(__floats2half2_rn(y[2], y[3])));
        // O^T: lane (g, t) has dims D/8 g .. of keys 2t, 2t + 1, 2t + 8, 2t + 9
        uint32_t v[4][kWords / 2];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = 2 * t + (r & 1) + 8 * (r >> 1);
            if constexpr (D == 128) {
                const uint4 x = lds128(vs + 16 * Shape::slot(row, g));
                v[r][0] = x.x, v[r][1] = x.y, v[r][2] = x.z, v[r][3] = x.w;
            } else {
                const uint2 x = lds64(vs + 16 * Shape::slot(row, g >> 1) + 8 * (g & 1));
                v[r][0] = x.x, v[r][1] = x.y;
            }
        }
#pragma unroll
        for (int w = 0; w < kWords / 2; ++w) {
            uint32_t a0, a1, a2, a3;
            unpack_word(__byte_perm(v[0][w], v[1][w], 0x5410), a0, a1);  // dim 4w: keys 2t, 2t + 1; dim 4w + 1
            unpack_word(__byte_perm(v[2][w], v[3][w], 0x5410), a2, a3);
            mma16816(o[2 * w], a0, a1, a2, a3, b0, b1);
            unpack_word(__byte_perm(v[0][w], v[1][w], 0x7632), a0, a1);  // dims 4w + 2, 4w + 3
            unpack_word(__byte_perm(v[2][w], v[3][w], 0x7632), a2, a3);
            mma16816(o[2 * w + 1], a0, a1, a2, a3, b0, b1);
        }
        __syncwarp();  // the stage is read before it is refilled
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], d);
        if (g == 0) {
            st_m[warp][2 * t + e] = m[e];
            st_l[warp][2 * t + e] = l[e];
        }
    }
    __syncthreads();  // every warp is done with its ring
    // ---- the CTA's O [8 heads][D]: each warp's share at its own reference, summed by dim
    constexpr int kPitch = D + 4;  // floats per (warp, head) row
    float *part = reinterpret_cast<float *>(smem);
    if (threadIdx.x < 8) {
        float top = kRefStart, sum = 0.0f;
        for (int w = 0; w < kDWarps; ++w) top = fmaxf(top, st_m[w][threadIdx.x]);
        for (int w = 0; w < kDWarps; ++w) sum += st_l[w][threadIdx.x] * exp2_approx(st_m[w][threadIdx.x] - top);
        cta_m[threadIdx.x] = top;
        cta_l[threadIdx.x] = sum;
    }
    __syncthreads();
    const float f0 = exp2_approx(m[0] - cta_m[2 * t]), f1 = exp2_approx(m[1] - cta_m[2 * t + 1]);
#pragma unroll
    for (int w = 0; w < kWords; ++w) {
        const int d = D / 8 * g + 2 * w;
        float *r0 = part + (warp * 8 + 2 * t) * kPitch + d, *r1 = r0 + kPitch;
        *reinterpret_cast<float2 *>(r0) = make_float2(o[w][0] * f0, o[w][2] * f0);
        *reinterpret_cast<float2 *>(r1) = make_float2(o[w][1] * f1, o[w][3] * f1);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 8 * D; i += kDThreads) {
        float *r = part + (i / D) * kPitch + i % D;
        float sum = r[0];
        for (int w = 1; w < kDWarps; ++w) sum += r[w * 8 * kPitch];
        r[0] = sum;
    }
    if (p.join) {
        float *dst = p.parts + ((static_cast<int64_t>(b) * gridDim.y + blockIdx.y) * p.splits + split) * 8 * (D + 2);
        __syncthreads();
        for (int i = threadIdx.x; i < heads * D; i += kDThreads) dst[i] = part[(i / D) * kPitch + i % D];
        if (threadIdx.x < heads) {
            dst[8 * D + threadIdx.x] = cta_m[threadIdx.x];
            dst[8 * D + 8 + threadIdx.x] = cta_l[threadIdx.x];
        }
        return;
    }
    // ---- the cluster's CTAs hold all of the sequence's keys: join through distributed shared memory
    cluster.sync();
    const int C = p.splits;
    if (threadIdx.x < 8) {
        float top = kRefStart, sum = 0.0f;
        for (int r = 0; r < C; ++r) top = fmaxf(top, *cluster.map_shared_rank(&cta_m[threadIdx.x], r));
        for (int r = 0; r < C; ++r)
            sum += *cluster.map_shared_rank(&cta_l[threadIdx.x], r) *
                   exp2_approx(*cluster.map_shared_rank(&cta_m[threadIdx.x], r) - top);
        st_m[0][threadIdx.x] = top;
        st_l[0][threadIdx.x] = sum;
        lse2[threadIdx.x] = top + log2f(sum);
    }
    __syncthreads();
    for (int i = split * kDThreads + threadIdx.x; i < heads * D; i += C * kDThreads) {
        const int h = i / D, d = i % D;
        float sum = 0.0f;
        for (int r = 0; r < C; ++r)
            sum = fmaf(*cluster.map_shared_rank(part + h * kPitch + d, r),
                       exp2_approx(*cluster.map_shared_rank(&cta_m[h], r) - st_m[0][h]), sum);
        a.out[b * a.o_sb + (h0 + h) * a.o_sh + d] = __float2half(n > 0 ? sum / st_l[0][h] : 0.0f);
    }
    if (a.lse && split == 0 && threadIdx.x < heads)
        a.lse[static_cast<int64_t>(b) * a.NH + h0 + threadIdx.x] = n > 0 ? lse2[threadIdx.x] * 0.6931471805599453f : -INFINITY;
    if (p.w_out) {
        for (int64_t key = k0 + threadIdx.x; key < k1; key += kDThreads) {
            const int64_t at = b * p.w_sb + head * p.w_sh + key;
            const float sum = key_weight(xs + key * group, lse2, group);
            p.w_out[at] = sum + (p.w_in && key < n - 1 ? p.w_in[at] : 0.0f);
        }
    }
    cluster.sync();  // no CTA leaves while another may read its shared memory
}

// Joins the splits of a (sequence, KV head).  Blocks 0 .. group - 1: one head's output, the splits dealt to the
// block's quarters; the others: the weights of 1024 keys each.
constexpr int kJoinThreads = 512;

template <int D>
__global__ void __launch_bounds__(kJoinThreads) attn8_join_kernel(DecodeArgs p) {
    extern __shared__ float sm[];  // [heads][splits] factors
    __shared__ float ref[128], sum[128], quarter[kJoinThreads];
    const AttnArgs &a = p.a;
    const int head = blockIdx.y, b = blockIdx.z, group = a.NH / a.pg.n_kv;
    const bool is_out = static_cast<int>(blockIdx.x) < group;
    pdl_wait();
    pdl_trigger();
    const int64_t n = visible(a.positions, b, 0, a.max_len);
    const int64_t w0 = (static_cast<int64_t>(blockIdx.x) - group) * 1024;
    if (!is_out && w0 >= n) return;
    constexpr int64_t kPart = 8 * (D + 2);
    const float *base = p.parts + (static_cast<int64_t>(b) * a.pg.n_kv + head) * p.head_chunks * p.splits * kPart;
    const int lane = threadIdx.x & 31;
    const int first = is_out ? blockIdx.x : 0, last = is_out ? first + 1 : group;
    for (int h = first + (threadIdx.x >> 5); h < last; h += kJoinThreads / 32) {
        const float *st = base + static_cast<int64_t>(h >> 3) * p.splits * kPart + 8 * D + (h & 7);
        float top = kRefStart, s = 0.0f;
        for (int i = lane; i < p.splits; i += 32) top = fmaxf(top, st[i * kPart]);
        top = warp_max(top);
        for (int i = lane; i < p.splits; i += 32) {
            const float f = exp2_approx(st[i * kPart] - top);
            sm[(h - first) * p.splits + i] = f;
            s = fmaf(st[i * kPart + 8], f, s);
        }
        s = warp_sum(s);
        if (lane == 0) ref[h - first] = top + log2f(s), sum[h - first] = s;
    }
    __syncthreads();
    if (!is_out) {
        const float *xs = p.scores + ((static_cast<int64_t>(b) * a.pg.n_kv + head) * p.s_len) * group;
        for (int64_t key = w0 + threadIdx.x; key < w0 + 1024 && key < n; key += kJoinThreads) {
            const int64_t at = b * p.w_sb + head * p.w_sh + key;
            const float w = key_weight(xs + key * group, ref, group);
            p.w_out[at] = w + (p.w_in && key < n - 1 ? p.w_in[at] : 0.0f);
        }
        return;
    }
    constexpr int kShare = kJoinThreads / D;
    const int d = threadIdx.x % D, q = threadIdx.x / D, h = first;
    const float *src = base + static_cast<int64_t>(h >> 3) * p.splits * kPart + (h & 7) * D + d;
    float acc = 0.0f;
#pragma unroll 8
    for (int s = q; s < p.splits; s += kShare) acc = fmaf(src[s * kPart], sm[s], acc);
    quarter[threadIdx.x] = acc;
    __syncthreads();
    if (threadIdx.x < D) {
        for (int i = 1; i < kShare; ++i) acc += quarter[i * D + d];
        a.out[b * a.o_sb + (head * group + h) * a.o_sh + d] = __float2half(n > 0 ? acc / sum[0] : 0.0f);
        if (a.lse && d == 0)
            a.lse[static_cast<int64_t>(b) * a.NH + head * group + h] = n > 0 ? ref[0] * 0.6931471805599453f : -INFINITY;
    }
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

struct DecodePlan {
    int splits, head_chunks;
    bool join;
    int64_t part_floats, floats;
};

// CTAs per sequence and head: four per SM in all, but at least 64 keys each and at most 2048.  Up to 8 join within
// their cluster; more (and groups of more than 8 heads whose weights are wanted, which no one CTA holds) in a
// second kernel.
DecodePlan decode_plan(int64_t B, int64_t NH, int64_t NK, int64_t D, int64_t max_len, int64_t splits, bool weights) {
    DecodePlan r = {};
    const int64_t group = NH / NK;
    r.head_chunks = static_cast<int>((group + 7) / 8);
    const int64_t units = B * NK * r.head_chunks;
    int64_t s = splits;
    if (s == 0) {
        s = 4 * sm_count() / units;
        const int64_t most = (max_len + 63) / 64, least = (max_len + 2047) / 2048;
        s = s < least ? least : s;
        s = s > most ? most : s;
    }
    const int64_t bound = 10240 / group;  // the joining kernel's shared memory
    s = s > 128 ? 128 : s;
    s = s > bound ? bound : s;
    s = s < 1 ? 1 : s;
    r.splits = static_cast<int>(s);
    r.join = s > 8 || (weights && r.head_chunks > 1);
    r.part_floats = r.join ? units * s * 8 * (D + 2) : 0;  // a multiple of 4: the scores behind stay aligned
    r.floats = r.part_floats + (weights ? B * NK * max_len * group : 0);
    return r;
}

template <typename Kernel>
int configure(Kernel kern, int smem, int slot, const char *what) {
    static bool done[16][64] = {};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) dev = 0;
    if (!done[slot][dev]) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
            return set_error(T2C_ECUDA, "%s: cudaFuncSetAttribute failed", what);
        done[slot][dev] = true;
    }
    return T2C_OK;
}

}  // namespace

cudaError_t status_attn8(unsigned int *bits, int clear, cudaStream_t s) { return read_tu_status(bits, clear, s); }

}  // namespace t2c

using namespace t2c;

extern "C" int64_t t2c_attn_decode_q8_workspace(const t2c_q8_pages *pages, int64_t bt_width, int64_t B, int64_t NH,
                                                int64_t max_len, int64_t splits, int with_weights) {
    if (!pages || pages->n_kv <= 0 || NH <= 0 || NH % pages->n_kv || B <= 0 || splits < 0 || bt_width <= 0) return -1;
    const int64_t capacity = bt_width * pages->page_size;
    if (max_len <= 0 || max_len > capacity) max_len = capacity;
    return decode_plan(B, NH, pages->n_kv, pages->head_dim, max_len, splits, with_weights != 0).floats;
}

extern "C" int t2c_attn_decode_q8(const t2c_q8_pages *pages, const void *q, int64_t q_sb, int64_t q_sh, void *out,
                                  int64_t o_sb, int64_t o_sh, float *lse, const int32_t *positions,
                                  const int32_t *block_table, int64_t bt_stride, int64_t bt_width, int64_t B, int64_t NH,
                                  float scale, int64_t max_len, int64_t splits, const float *weights, float *weights_out,
                                  int64_t w_sb, int64_t w_sh, float *workspace, int64_t workspace_floats, void *stream) {
    DecodeArgs p = {};
    AttnArgs &a = p.a;
    int rc = check(pages, "attn_decode_q8", a.pg, block_table, bt_stride, bt_width, positions, B, 1, NH, max_len);
    if (rc != T2C_OK) return rc;
    if (!strides_ok(q, q_sb, q_sh, 0) || !strides_ok(out, o_sb, o_sh, 0))
        return set_error(T2C_EINVAL, "attn_decode_q8: q and out rows must be 16-byte aligned");
    if (splits < 0) return set_error(T2C_EINVAL, "attn_decode_q8: splits %lld", (long long)splits);
    const int64_t D = pages->head_dim, group = NH / a.pg.n_kv;
    if (group > 128) return set_error(T2C_EUNSUPPORTED, "attn_decode_q8: group %lld", (long long)group);
    const DecodePlan plan = decode_plan(B, NH, a.pg.n_kv, D, max_len, splits, weights_out != nullptr);
    if (plan.floats > 0 && (!workspace || workspace_floats < plan.floats))
        return set_error(T2C_ESCRATCH, "attn_decode_q8: workspace needs %lld floats", (long long)plan.floats);
    if (!kv8_aligned(workspace, 16)) return set_error(T2C_EINVAL, "attn_decode_q8: workspace must be 16-byte aligned");
    if (a.pg.n_kv * plan.head_chunks > 65535) return set_error(T2C_EINVAL, "attn_decode_q8: bad shape");
    a.q = static_cast<const __half *>(q), a.q_sb = q_sb, a.q_sh = q_sh;
    a.out = static_cast<__half *>(out), a.o_sb = o_sb, a.o_sh = o_sh;
    a.lse = lse;
    a.positions = positions, a.table = block_table, a.t_stride = bt_stride, a.max_len = max_len;
    a.B = static_cast<int>(B), a.T = 1, a.NH = static_cast<int>(NH);
    a.scale_log2 = scale * 1.4426950408889634f;
    p.splits = plan.splits, p.head_chunks = plan.head_chunks, p.join = plan.join;
    p.parts = workspace;
    p.scores = workspace + plan.part_floats;
    p.s_len = max_len;
    p.w_in = weights, p.w_out = weights_out, p.w_sb = w_sb, p.w_sh = w_sh;
    const cudaStream_t s = as_stream(stream);
    const auto kern = D == 128 ? attn8_decode_kernel<128> : attn8_decode_kernel<64>;
    const int smem = D == 128 ? DecodeShape<128>::kRing : DecodeShape<64>::kRing;
    rc = configure(kern, smem, D == 128 ? 0 : 1, "attn_decode_q8");
    if (rc != T2C_OK) return rc;
    rc = kv8_launch("attn_decode_q8", kern,
                    dim3(static_cast<unsigned>(p.splits), static_cast<unsigned>(a.pg.n_kv * p.head_chunks), static_cast<unsigned>(B)),
                    dim3(kDThreads), smem, p.join ? 1u : static_cast<unsigned>(p.splits), s, p);
    if (rc != T2C_OK || !p.join) return rc;
    const int64_t chunks = weights_out ? (max_len + 1023) / 1024 : 0;
    return kv8_launch("attn_decode_q8 join", D == 128 ? attn8_join_kernel<128> : attn8_join_kernel<64>,
                      dim3(static_cast<unsigned>(group + chunks), static_cast<unsigned>(a.pg.n_kv), static_cast<unsigned>(B)),
                      dim3(kJoinThreads), static_cast<size_t>((weights_out ? group : 1) * p.splits * 4), 1, s, p);
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
