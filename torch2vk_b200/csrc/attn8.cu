// Attention of single tokens over the paged KV cache in 8 bits.
#include <cooperative_groups.h>
#include <cudaTypedefs.h>

#include <type_traits>

#include "kv8.cuh"
#include "kv8_parts.cuh"

namespace cg = cooperative_groups;

namespace t2c {
namespace {

struct AttnArgs {
    KvPages pg;
    const __half *q;
    int64_t q_sb, q_sh;
    __half *out;
    int64_t o_sb, o_sh;
    float *lse;  // [B, NH]
    const int32_t *positions, *table;
    int64_t t_stride, max_len;
    int B, NH;
    float scale_log2;
};

// Number of keys the query of sequence b sees.
__device__ __forceinline__ int64_t visible(const int32_t *positions, int b, int64_t max_len) {
    const int64_t n = static_cast<int64_t>(positions[b]) + 1;
    if (n > max_len) {
        report_device_error(T2C_EINVAL);
        return max_len;
    }
    return n < 0 ? 0 : n;
}

// ------------------------------------------------------------------ one token per sequence
// Work is cut into tiles of 64 keys of one (sequence, KV head, 8 heads of the group); a fixed number of CTAs takes
// equal runs of the list of tiles (whatever the sequences' lengths), so a run covers the end of one unit, whole
// units, and the beginning of another: units that a CTA covers wholly it finishes itself, the others a second kernel
// joins.  Short caches take one cluster per unit instead, joined in distributed shared memory by the same launch.
// Inside a CTA a warp takes every fourth 16 keys, in a ring of kDStages steps of its own: TMA boxes of 16 rows
// (swizzled, so that the fragment reads below hit each bank once), one mbarrier per stage, no CTA barrier in the
// loop.  16 keys lie in one block of the cache, so one K and one V scale serve a step.  Both products run on
// mma.m16n8k16 with the heads as the n side, so that a cached byte is expanded once for all heads of the group:
//   S^T [16 keys x 8 heads] = K Q^T,   O^T [16 dims x 8 heads] += V^T P^T.
// Codes become fp16 exactly.  The scales stay in fp32: x = s * (k scale * softmax scale * log2 e), and the V scale
// joins the exponent, P = 2^(x + log2 vs - m), so that P q_v needs no scaled V; the softmax sum takes P / vs.  m is a
// running reference per head, moved (and O, l rescaled) only when some exponent passes 14: P stays in fp16's range,
// and its one rounding to fp16, which the tensor core asks for, is the only one before the output's.
// What bounds it: the cache's bytes where there are many (32 sequences of up to 6007 positions, 32 heads of 128 on 8:
// 251 MB in 49 us, 5.1 TB/s; with the weights 259 MB in 58 us), the chain of a CTA's beginning, its few tiles and the
// join where there are few (32801 positions of one sequence: 67 MB in 24 us, 7 of them the join).  Two steps of ring, four
// CTAs an SM: with three or four steps, or eight warps, fewer CTAs fit and the time with the weights was 5 % longer.
constexpr int kDWarps = 4;
constexpr int kDStages = 2;
constexpr int kDThreads = 32 * kDWarps;
constexpr int kDTile = 16 * kDWarps;
constexpr float kRefStart = -1e30f;  // below any finite score: the first step moves it
constexpr float kRefTop = 14.0f;     // P <= 2^14
constexpr float kRefDrop = 8.0f;     // a moved reference leaves the largest P at 2^8

template <int D>
struct DecodeShape {
    static constexpr int kStep = 16 * D;  // bytes of K (or V) per step
    static constexpr int kRing = kDWarps * kDStages * 2 * kStep;
    static constexpr int kPart = 8 * (D + 2);  // floats of a partial result: O, m, l of 8 heads
    // byte offset of 16-byte chunk c of row r in a TMA box (128- or 64-byte swizzle); chunk c + 2 j is at ^ (32 j)
    static __device__ __forceinline__ uint32_t at(int r, int c) {
        return static_cast<uint32_t>(D == 128 ? r * 128 + ((c ^ (r & 7)) << 4) : r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
    }
};

// Four 8 x 16-byte tiles, a row's address from each lane: lane (g, t) gets bytes 4t .. 4t + 3 of each tile's row g, or
// transposed by byte pairs: bytes 2g, 2g + 1 of rows 2t and 2t + 1.
__device__ __forceinline__ void ldsm(uint32_t v[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "r"(a)
                 : "memory");
}
__device__ __forceinline__ void ldsm_trans(uint32_t v[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                 : "r"(a)
                 : "memory");
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
    int splits;       // CTAs per unit in a cluster; 0: tile runs, joined by the second kernel
    int head_chunks;  // chunks of 8 heads of a group
    int ctas;         // of the tile runs
    int most_parts;   // of a unit
    float *parts;     // [2 * ctas][kPart]
    int2 *unit_ctas;  // [B * n_kv * head_chunks] first and last CTA of a unit's tiles
    float *unit_lse;  // [B][NH] in log2 units, of units one CTA finished; where the weights are wanted
    float *scores;    // [B][n_kv][s_len][group] x in log2 units, where the weights are wanted
    int64_t s_len;
    const float *w_in;
    float *w_out;
    int64_t w_sb, w_sh;
};

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

// Tiles of sequence b: an empty sequence keeps one, whose CTA writes its zeros.
__device__ __forceinline__ int seq_tiles(const AttnArgs &a, int b) {
    const int64_t n = min(static_cast<int64_t>(a.positions[b]) + 1, a.max_len);
    return n <= kDTile ? 1 : static_cast<int>((n + kDTile - 1) / kDTile);
}

template <int D>
__global__ void __launch_bounds__(kDThreads, 4) attn8_decode_kernel(const __grid_constant__ CUtensorMap k_map,
                                                                    const __grid_constant__ CUtensorMap v_map,
                                                                    const __grid_constant__ DecodeArgs p) {
    using Shape = DecodeShape<D>;
    constexpr int kWords = D / 16;  // K: 32-bit words per lane and row = k steps; V: m tiles
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ uint64_t full[kDWarps][kDStages];
    __shared__ float4 metas[kDWarps][64];  // of two windows of 32 steps: K factor, log2 V scale, 1 / V scale, page
    __shared__ float st_m[kDWarps][8], st_l[kDWarps][8], cta_m[8], cta_l[8], lse2[8];
    const AttnArgs &a = p.a;
    cg::cluster_group cluster = cg::this_cluster();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int group = a.NH / a.pg.n_kv;
    const int units = a.pg.n_kv * p.head_chunks;  // of a sequence
    if (threadIdx.x < kDWarps * kDStages) mbar_init(&full[0][0] + threadIdx.x, 1);
    fence_mbar_init();
    __syncthreads();
    if (smem_u32(smem) & 1023u) {  // the swizzle needs it: report, compute nothing
        if (threadIdx.x == 0) report_device_error(T2C_EUNSUPPORTED);
        return;
    }
    pdl_wait();
    pdl_trigger();

    // ---- this CTA's tiles: of its cluster's unit, or its run of all tiles
    int b = 0, unit = 0, t0 = 0, left = 0, unit_tiles = 1;
    if (p.splits > 0) {
        b = blockIdx.z, unit = blockIdx.y;
        unit_tiles = seq_tiles(a, b);
        const int per = (unit_tiles + p.splits - 1) / p.splits;
        t0 = min(per * static_cast<int>(blockIdx.x), unit_tiles);
        left = min(per, unit_tiles - t0);
    } else {
        int total = 0;
        for (int i = lane; i < a.B; i += 32) total += seq_tiles(a, i);
        total = units * __reduce_add_sync(0xffffffffu, total);
        const int ctas = min(p.ctas, total);  // each has a tile or more
        const int c = blockIdx.x;
        if (c >= ctas) return;
        const int per = total / ctas, extra = total % ctas;
        const int from = c * per + min(c, extra);
        left = per + (c < extra ? 1 : 0);
        // 32 sequences at a time: the one that holds tile `from`
        int before = 0;
        for (int base = 0; base < a.B; base += 32) {
            const int mine = base + lane < a.B ? units * seq_tiles(a, base + lane) : 0;
            int incl = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += v;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, before + incl > from);
            if (past) {
                const int i = __ffs(past) - 1;
                b = base + i;
                unit_tiles = __shfl_sync(0xffffffffu, mine, i) / units;
                const int local = from - (before + __shfl_sync(0xffffffffu, incl - mine, i));
                unit = local / unit_tiles;
                t0 = local % unit_tiles;
                break;
            }
            before += __shfl_sync(0xffffffffu, incl, 31);
        }
    }

    const uint32_t ring = smem_u32(smem) + warp * (kDStages * 2 * Shape::kStep);
    const int page_mask = (1 << a.pg.page_log2) - 1;
    const uint32_t frag = Shape::at(lane & 15, lane >> 4);  // the lane's row of a fragment load: 16 rows, 2 chunks
    uint32_t phases = 0;  // of this warp's stages
    bool failed = false;
    do {
        const int head = unit / p.head_chunks, chunk = unit % p.head_chunks;
        const int heads = min(8, group - 8 * chunk), h0 = head * group + 8 * chunk;
        const int64_t n = visible(a.positions, b, a.max_len);
        const int t1 = min(t0 + left, unit_tiles);
        const int64_t k0 = min(static_cast<int64_t>(t0) * kDTile, n), k1 = min(static_cast<int64_t>(t1) * kDTile, n);
        const int32_t *bt = a.table + b * a.t_stride;
        const int steps = static_cast<int>((k1 - k0 + 15) >> 4);                     // of the CTA
        const int mine = steps > warp ? (steps - warp + kDWarps - 1) / kDWarps : 0;  // of this warp: warp, warp + 4, ..
        const auto step_key = [&](int i) { return k0 + 16 * warp + static_cast<int64_t>(kDTile) * i; };
        float4 *meta = metas[warp];

        // pages and scales of 32 steps: page, then scales, then the factors, each a few steps after the one before
        int next_page = 0;
        __half next_ks, next_vs;
        const auto look_page = [&](int window) {
            const int i = window * 32 + lane;
            next_page = i < mine ? max(kv8_page(a.pg, bt, step_key(i)), 0) : 0;
        };
        const auto look_scales = [&](int window) {
            const int i = window * 32 + lane;
            const int64_t so = i < mine ? kv8_scale_offset(a.pg, next_page, head, step_key(i)) : 0;
            next_ks = a.pg.ks[so];
            next_vs = a.pg.vs[so];
        };
        bool nan_values = false;  // a V block of this lane's steps reads as NaN
        const auto store_meta = [&](int window) {
            const float vs = __half2float(next_vs);
            // a block of scale 0 has values 0: any exponent adds nothing to O, the least scale's moves no reference.  One of
            // NaN is taken alike, so that the softmax's statistics, which are the scores' alone, stay theirs; O becomes NaN
            // at the end.
            const bool flat = vs == 0.0f || vs != vs;
            nan_values |= vs != vs && window * 32 + lane < mine;
            meta[(window & 1) * 32 + lane] =
                make_float4(__half2float(next_ks) * a.scale_log2, flat ? -24.0f : log2f(vs),
                            flat ? 16777216.0f : 1.0f / vs, __int_as_float(next_page));
            __syncwarp();
        };
        const auto load = [&](int i, int stage, int page) {  // by one lane
            const uint32_t st = ring + stage * 2 * Shape::kStep;
            mbar_arrive_expect_tx(&full[warp][stage], 2 * Shape::kStep);
            const int row = static_cast<int>(step_key(i)) & page_mask;
            tma_load_4d(st, &k_map, 0, row, head, page, &full[warp][stage]);
            tma_load_4d(st + Shape::kStep, &v_map, 0, row, head, page, &full[warp][stage]);
        };
        look_page(0);
#pragma unroll
        for (int i = 0; i < kDStages; ++i) {
            const int page = __shfl_sync(0xffffffffu, next_page, i);
            if (lane == 0 && i < mine) load(i, i, page);
        }
        look_scales(0);

        // ---- Q^T fragments: k step i, lane (g, t): head g, dims 16 i + 4 t + {0, 2} and {1, 3}
        uint32_t qf[kWords][2];
        {
            const uint32_t *q = reinterpret_cast<const uint32_t *>(a.q + b * a.q_sb + (h0 + min(g, heads - 1)) * a.q_sh) + 2 * t;
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                const uint32_t lo = g < heads ? q[8 * i] : 0u, hi = g < heads ? q[8 * i + 1] : 0u;
                qf[i][0] = __byte_perm(lo, hi, 0x5410);
                qf[i][1] = __byte_perm(lo, hi, 0x7632);
            }
        }
        store_meta(0);

        float o[kWords][4] = {};
        float m[2] = {kRefStart, kRefStart}, l[2] = {0.0f, 0.0f};
        float *xs = p.scores + ((static_cast<int64_t>(b) * a.pg.n_kv + head) * p.s_len) * group + 8 * chunk;
        float *xp = xs + (k0 + 16 * warp + g) * group + 2 * t;
        int rem = static_cast<int>(k1 - k0) - 16 * warp - g;  // keys from this lane's first one to the end
#pragma unroll 1
        for (int i0 = 0; i0 < mine && !failed; i0 += kDStages) {
#pragma unroll
            for (int st = 0; st < kDStages; ++st) {
                const int i = i0 + st;
                if (i >= mine) break;
                if ((i | 31) + 1 < mine) {  // the next window's look-ups, spread over this one's steps
                    const int at = i & 31;
                    if (at == 4) look_page(i / 32 + 1);
                    if (at == 12) look_scales(i / 32 + 1);
                    if (at == 20) store_meta(i / 32 + 1);
                }
                const bool arrived = mbar_wait(&full[warp][st], (phases >> st) & 1u);
                if (!__all_sync(0xffffffffu, arrived)) {
                    // the copies of this step and of those loaded ahead end (or are given up) before the CTA may
                    for (int k = 0; k < kDStages && i + k < mine; ++k)
                        mbar_wait(&full[warp][(st + k) % kDStages], (phases >> ((st + k) % kDStages)) & 1u);
                    failed = true;
                    break;
                }
                phases ^= 1u << st;
                const float4 f = meta[i & 63];
                const uint32_t ks = ring + st * 2 * Shape::kStep, vs = ks + Shape::kStep;
                // S^T: 16 dims a k step; two chains
                float s[4] = {}, s2[4] = {};
#pragma unroll
                for (int c = 0; c < kWords; c += 2) {
                    uint32_t w[4], a0, a1, a2, a3;
                    ldsm(w, ks + (frag ^ (16 * c)));
                    unpack_word(w[0], a0, a2);
                    unpack_word(w[1], a1, a3);
                    mma16816(s, a0, a1, a2, a3, qf[c][0], qf[c][1]);
                    unpack_word(w[2], a0, a2);
                    unpack_word(w[3], a1, a3);
                    mma16816(s2, a0, a1, a2, a3, qf[c + 1][0], qf[c + 1][1]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) s[e] += s2[e];
                // s[0], s[1]: key g, heads 2t, 2t + 1; s[2], s[3]: key g + 8
                const bool in0 = rem > 0, in1 = rem > 8;
                if (p.w_out) {
                    if (in0 && 2 * t < heads) xp[0] = s[0] * f.x;
                    if (in0 && 2 * t + 1 < heads) xp[1] = s[1] * f.x;
                    if (in1 && 2 * t < heads) xp[8 * group] = s[2] * f.x;
                    if (in1 && 2 * t + 1 < heads) xp[8 * group + 1] = s[3] * f.x;
                    xp += kDTile * group;
                }
                rem -= kDTile;
                float y[4];
                y[0] = in0 ? fmaf(s[0], f.x, f.y - m[0]) : -INFINITY;
                y[1] = in0 ? fmaf(s[1], f.x, f.y - m[1]) : -INFINITY;
                y[2] = in1 ? fmaf(s[2], f.x, f.y - m[0]) : -INFINITY;
                y[3] = in1 ? fmaf(s[3], f.x, f.y - m[1]) : -INFINITY;
                if (__any_sync(0xffffffffu, fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])) > kRefTop)) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float top = fmaxf(in0 ? fmaf(s[e], f.x, f.y) : -INFINITY, in1 ? fmaf(s[2 + e], f.x, f.y) : -INFINITY);
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
                        y[e] = in0 ? fmaf(s[e], f.x, f.y - ref) : -INFINITY;
                        y[2 + e] = in1 ? fmaf(s[2 + e], f.x, f.y - ref) : -INFINITY;
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = exp2_approx(y[e]);
                l[0] = fmaf(y[0] + y[2], f.z, l[0]);
                l[1] = fmaf(y[1] + y[3], f.z, l[1]);
                const uint32_t b0 = transpose8x8(half2_bits(__floats2half2_rn(y[0], y[1])));
                const uint32_t b1 = transpose8x8(half2_bits(__floats2half2_rn(y[2], y[3])));
                // O^T: m tile c, lane (g, t): dims 16 c + 2 g + {0, 1} of keys 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
                for (int c = 0; c < kWords; c += 2) {
                    uint32_t w[4], a0, a1, a2, a3;
                    ldsm_trans(w, vs + (frag ^ (16 * c)));
                    unpack_word(w[0], a0, a1);
                    unpack_word(w[1], a2, a3);
                    mma16816(o[c], a0, a1, a2, a3, b0, b1);
                    unpack_word(w[2], a0, a1);
                    unpack_word(w[3], a2, a3);
                    mma16816(o[c + 1], a0, a1, a2, a3, b0, b1);
                }
                __syncwarp();  // the stage is read before it is refilled
                if (lane == 0 && i + kDStages < mine)
                    load(i + kDStages, st, __float_as_int(meta[(i + kDStages) & 63].w));
            }
        }
        if (__any_sync(0xffffffffu, nan_values)) {
#pragma unroll
            for (int w = 0; w < kWords; ++w) o[w][0] = o[w][1] = o[w][2] = o[w][3] = __int_as_float(0x7fffffff);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], d);
            if (g == 0) {
                st_m[warp][2 * t + e] = m[e];
                st_l[warp][2 * t + e] = l[e];
            }
        }
        failed = __syncthreads_or(failed);  // every warp is done with its ring
        if (failed) {
            if (threadIdx.x == 0) report_device_error(T2C_ETIMEOUT);
            break;
        }
        // ---- the CTA's O [8 heads][D]: each warp's share at the common reference, summed
        constexpr int kPitch = D + 4;  // floats per (warp, head) row
        float *part = reinterpret_cast<float *>(smem);
        if (threadIdx.x < 8) {
            float top = kRefStart, sum = 0.0f;
            for (int w = 0; w < kDWarps; ++w) top = fmaxf(top, st_m[w][threadIdx.x]);
            for (int w = 0; w < kDWarps; ++w) sum += st_l[w][threadIdx.x] * exp2_approx(st_m[w][threadIdx.x] - top);
            cta_m[threadIdx.x] = top;
            cta_l[threadIdx.x] = sum;
            lse2[threadIdx.x] = top + log2f(sum);
        }
        {
            float top[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                top[e] = kRefStart;
                for (int w = 0; w < kDWarps; ++w) top[e] = fmaxf(top[e], st_m[w][2 * t + e]);
                top[e] = exp2_approx(m[e] - top[e]);
            }
#pragma unroll
            for (int w = 0; w < kWords; ++w) {
                const int d = 16 * w + 2 * g;
                float *r0 = part + (warp * 8 + 2 * t) * kPitch + d, *r1 = r0 + kPitch;
                *reinterpret_cast<float2 *>(r0) = make_float2(o[w][0] * top[0], o[w][2] * top[0]);
                *reinterpret_cast<float2 *>(r1) = make_float2(o[w][1] * top[1], o[w][3] * top[1]);
            }
        }
        __syncthreads();
        const bool whole = t0 == 0 && t1 == unit_tiles;  // and so finished here
        const bool shared = p.splits > 1;
        float *dst = p.parts + (2 * static_cast<int64_t>(blockIdx.x) + (t0 == 0 ? 1 : 0)) * Shape::kPart;
        for (int i = threadIdx.x; i < heads * D; i += kDThreads) {
            const int h = i / D, d = i % D;
            float *r = part + h * kPitch + d;
            float sum = r[0];
            for (int w = 1; w < kDWarps; ++w) sum += r[w * 8 * kPitch];
            if (shared)
                r[0] = sum;
            else if (whole)
                a.out[b * a.o_sb + (h0 + h) * a.o_sh + d] = __float2half(n > 0 ? sum / cta_l[h] : 0.0f);
            else
                dst[i] = sum;
        }
        if (!shared && threadIdx.x < heads) {
            const int64_t row = static_cast<int64_t>(b) * a.NH + h0 + threadIdx.x;
            if (whole) {
                if (a.lse) a.lse[row] = n > 0 ? lse2[threadIdx.x] * 0.6931471805599453f : -INFINITY;
                if (p.w_out && p.splits == 0) p.unit_lse[row] = lse2[threadIdx.x];
            } else {
                dst[8 * D + threadIdx.x] = cta_m[threadIdx.x];
                dst[8 * D + 8 + threadIdx.x] = cta_l[threadIdx.x];
            }
        }
        if (p.splits > 0) break;
        if (threadIdx.x == 0) {
            int2 *at = p.unit_ctas + static_cast<int64_t>(b) * units + unit;
            if (t0 == 0) at->x = blockIdx.x;
            if (t1 == unit_tiles) at->y = blockIdx.x;
        }
        // the next unit; its copies overwrite what the loop above read
        left -= t1 - t0;
        t0 = 0;
        if (++unit == units && left > 0) {
            unit = 0;
            ++b;
            unit_tiles = seq_tiles(a, b);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads();
    } while (left > 0);
    if (p.splits == 0) return;
    // ---- the cluster's CTAs hold all of the unit's keys: join through distributed shared memory
    const int head = unit / p.head_chunks, chunk = unit % p.head_chunks;
    const int heads = min(8, group - 8 * chunk), h0 = head * group + 8 * chunk;
    const int64_t n = visible(a.positions, b, a.max_len);
    const int C = p.splits;
    constexpr int kPitch = D + 4;
    float *part = reinterpret_cast<float *>(smem);
    if (C > 1) {
        cluster.sync();
        if (threadIdx.x < 8) {
            float top = kRefStart, sum = 0.0f;
            for (int r = 0; r < C; ++r) top = fmaxf(top, *cluster.map_shared_rank(&cta_m[threadIdx.x], r));
            for (int r = 0; r < C; ++r) {
                const float f = exp2_approx(*cluster.map_shared_rank(&cta_m[threadIdx.x], r) - top);
                sum += *cluster.map_shared_rank(&cta_l[threadIdx.x], r) * f;
                metas[r >> 2][8 * (r & 3) + threadIdx.x].x = f;  // factors [rank][head]
            }
            st_m[0][threadIdx.x] = sum;
            lse2[threadIdx.x] = top + log2f(sum);
        }
        __syncthreads();
        for (int i = blockIdx.x * kDThreads + threadIdx.x; i < heads * D; i += C * kDThreads) {
            const int h = i / D, d = i % D;
            float sum = 0.0f;
            for (int r = 0; r < C; ++r)
                sum = fmaf(*cluster.map_shared_rank(part + h * kPitch + d, r), metas[r >> 2][8 * (r & 3) + h].x, sum);
            a.out[b * a.o_sb + (h0 + h) * a.o_sh + d] = __float2half(n > 0 ? sum / st_m[0][h] : 0.0f);
        }
        if (a.lse && blockIdx.x == 0 && threadIdx.x < heads)
            a.lse[static_cast<int64_t>(b) * a.NH + h0 + threadIdx.x] =
                n > 0 ? lse2[threadIdx.x] * 0.6931471805599453f : -INFINITY;
    }
    if (p.w_out) {  // one chunk of heads: this CTA's own scores
        const float *xs = p.scores + ((static_cast<int64_t>(b) * a.pg.n_kv + head) * p.s_len) * group;
        const int64_t end = min(static_cast<int64_t>(t0 + left) * kDTile, n);
        for (int64_t key = static_cast<int64_t>(t0) * kDTile + threadIdx.x; key < end; key += kDThreads) {
            const int64_t at = b * p.w_sb + head * p.w_sh + key;
            const float sum = key_weight(xs + key * group, lse2, group);
            p.w_out[at] = sum + (p.w_in && key < n - 1 ? p.w_in[at] : 0.0f);
        }
    }
    if (C > 1) cluster.sync();  // no CTA leaves while another may read its shared memory
}

// Joins the runs.  The first blocks of a (sequence, KV head): the output of one head, its parts dealt to the block's
// quarters, or of a head for each quarter; the others: the weights of 4096 keys each.  What does not depend on the softmax statistics is loaded
// beside them: a block is three dependent trips to memory long (32801 positions of one sequence: 7 us; 32 sequences of up to
// 6007 with the weights: 10 us, 8 MB).
constexpr int kJoinThreads = 512;
constexpr int kJoinKeys = 4096;

template <int D, bool ALONE>
__global__ void __launch_bounds__(kJoinThreads) attn8_join_kernel(const __grid_constant__ DecodeArgs p) {
    constexpr int kShare = kJoinThreads / D, kHeads = ALONE ? 1 : kShare, kAhead = 4;
    extern __shared__ float factor[];  // [parts] of the block's heads
    __shared__ float ref[128], sum[kShare], quarter[kJoinThreads];
    constexpr int kPart = DecodeShape<D>::kPart;
    const AttnArgs &a = p.a;
    const int head = blockIdx.y, b = blockIdx.z, group = a.NH / a.pg.n_kv;
    const int out_blocks = (group + kHeads - 1) / kHeads;
    const bool is_out = static_cast<int>(blockIdx.x) < out_blocks;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int2 *ctas = p.unit_ctas + (static_cast<int64_t>(b) * a.pg.n_kv + head) * p.head_chunks;
    const int first = is_out ? blockIdx.x * kHeads : 0, last = is_out ? min(first + kHeads, group) : group;
    const int64_t n = min(static_cast<int64_t>(a.positions[b]) + 1, a.max_len);
    const int64_t w0 = (static_cast<int64_t>(blockIdx.x) - out_blocks) * kJoinKeys;
    if (!is_out && w0 >= n) return;
    pdl_wait();  // positions were there before the kernel whose parts are joined
    pdl_trigger();
    const int2 own = ctas[first >> 3];
    const int count = kv8_part_count(own.x, own.y, p.ctas, p.most_parts);
    if (is_out && count <= 1) return;  // a unit of one CTA is written, one whose CTA gave up has no result
    // part i of a unit whose tiles begin in CTA c0: that CTA's last one, then the others' first
    const auto part_of = [&](int c0, int i) { return p.parts + (2 * static_cast<int64_t>(c0 + i) + (i == 0 ? 1 : 0)) * kPart; };

    // a quarter: every kShare-th part of the block's head, or all parts of its own head
    const int d = threadIdx.x % D, q = threadIdx.x / D;
    const int mine = ALONE ? first : min(first + q, group - 1), part0 = ALONE ? q : 0;
    constexpr int step = ALONE ? kShare : 1;
    float ahead[kAhead];
    if (is_out) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            ahead[k] = part0 + step * k < count ? part_of(own.x, part0 + step * k)[(mine & 7) * D + d] : 0.0f;
    }
    for (int h = first + warp; h < last; h += kJoinThreads / 32) {
        const int2 c = ctas[h >> 3];
        const int parts = kv8_part_count(c.x, c.y, p.ctas, p.most_parts);
        if (parts <= 1) {  // without a result: no probability
            if (lane == 0) ref[h] = parts == 1 ? p.unit_lse[static_cast<int64_t>(b) * a.NH + head * group + h] : INFINITY;
            continue;
        }
        float top = kRefStart, s = 0.0f, m0 = kRefStart, l0 = 0.0f;
        if (lane < parts) {
            const float *st = part_of(c.x, lane) + 8 * D + (h & 7);
            top = m0 = st[0];
            l0 = st[8];
        }
        for (int i = lane + 32; i < parts; i += 32) top = fmaxf(top, part_of(c.x, i)[8 * D + (h & 7)]);
        top = warp_max(top);
        for (int i = lane; i < parts; i += 32) {
            const float *st = part_of(c.x, i) + 8 * D + (h & 7);
            const float f = exp2_approx((i == lane ? m0 : st[0]) - top);
            if (is_out) factor[(h - first) * count + i] = f;
            s = fmaf(i == lane ? l0 : st[8], f, s);
        }
        s = warp_sum(s);
        if (lane == 0) {
            ref[h] = top + log2f(s);
            if (is_out) sum[h - first] = s;
        }
    }
    if (!is_out) {
        const float *xs = p.scores + ((static_cast<int64_t>(b) * a.pg.n_kv + head) * p.s_len + w0) * group;
        const int64_t at = b * p.w_sb + head * p.w_sh + w0;
        const int end = static_cast<int>(n - w0 < kJoinKeys ? n - w0 : kJoinKeys), old = static_cast<int>(n - 1 - w0);
        // scores of eight keys a thread, all in flight before the statistics are known
        const auto ahead_of = [&](auto heads) {
            constexpr int G = decltype(heads)::value, kKeys = kJoinKeys / kJoinThreads;
            using Vec = typename std::conditional<G == 4, float4, typename std::conditional<G == 2, float2, float>::type>::type;
            Vec x[kKeys];
            float w[kKeys];
#pragma unroll
            for (int k = 0; k < kKeys; ++k) {
                const int key = threadIdx.x + kJoinThreads * k;
                if (key < end) x[k] = *reinterpret_cast<const Vec *>(xs + G * key);
                w[k] = p.w_in && key < end && key < old ? p.w_in[at + key] : 0.0f;
            }
            __syncthreads();
            float r[G];
#pragma unroll
            for (int g = 0; g < G; ++g) r[g] = ref[g];
#pragma unroll
            for (int k = 0; k < kKeys; ++k) {
                const int key = threadIdx.x + kJoinThreads * k;
                const float *v = reinterpret_cast<const float *>(&x[k]);
                float total = 0.0f;
#pragma unroll
                for (int g = 0; g < G; ++g) total += exp2_approx(v[g] - r[g]);
                if (key < end) p.w_out[at + key] = w[k] + total;
            }
        };
        if (group == 4) return ahead_of(std::integral_constant<int, 4>{});
        if (group == 2) return ahead_of(std::integral_constant<int, 2>{});
        if (group == 1) return ahead_of(std::integral_constant<int, 1>{});
        __syncthreads();
        for (int key = threadIdx.x; key < end; key += kJoinThreads) {
            const float w = key_weight(xs + static_cast<int64_t>(key) * group, ref, group);
            p.w_out[at + key] = w + (p.w_in && key < old ? p.w_in[at + key] : 0.0f);
        }
        return;
    }
    __syncthreads();
    float acc = 0.0f;
    const float *f = factor + (ALONE ? 0 : (mine - first) * count);
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
        if (part0 + step * k < count) acc = fmaf(ahead[k], f[part0 + step * k], acc);
#pragma unroll 8
    for (int i = part0 + step * kAhead; i < count; i += step) acc = fmaf(part_of(own.x, i)[(mine & 7) * D + d], f[i], acc);
    if (ALONE) {
        quarter[threadIdx.x] = acc;
        __syncthreads();
        if (threadIdx.x >= D) return;
        for (int i = 1; i < kShare; ++i) acc += quarter[i * D + d];
    } else if (first + q >= last) {
        return;
    }
    a.out[b * a.o_sb + (head * group + mine) * a.o_sh + d] = __float2half(acc / sum[mine - first]);
    if (a.lse && d == 0) a.lse[static_cast<int64_t>(b) * a.NH + head * group + mine] = ref[mine] * 0.6931471805599453f;
}

struct DecodePlan {
    int splits, head_chunks, ctas;
    int64_t part_floats, unit_floats, lse_floats, floats;
};

// A cluster of one 64-key tile per CTA where the longest sequence has at most 8 tiles and one wave of CTAs holds
// them all (a group of more than 8 heads whose weights are wanted is in no one CTA's hands, so it takes the runs);
// else runs of tiles, four CTAs per SM.  (333 positions, 16 heads on 8: 6.7 us, as runs 7.1; 8 sequences of 512, 32 heads
// on 8: 8.1, 9.5; but 32 of them 31.7 as clusters, 15.3 as runs.)
DecodePlan decode_plan(int64_t B, int64_t NH, int64_t NK, int64_t D, int64_t max_len, int64_t splits, bool weights) {
    DecodePlan r = {};
    const int64_t group = NH / NK;
    r.head_chunks = static_cast<int>((group + 7) / 8);
    const int64_t units = B * NK * r.head_chunks, tiles = (max_len + kDTile - 1) / kDTile, wave = 4 * sm_count();
    if (splits == 0 && tiles <= 8 && units * tiles <= wave && !(weights && r.head_chunks > 1)) {
        r.splits = static_cast<int>(tiles);
    } else {
        const int64_t most = units * tiles;
        int64_t ctas = splits > 0 ? (splits < most / units ? splits * units : most) : (wave < most ? wave : most);
        r.ctas = static_cast<int>(ctas < 8192 ? ctas : 8192);
        r.part_floats = 2 * r.ctas * 8 * (D + 2);  // a multiple of 4: what lies behind stays aligned
        r.unit_floats = (2 * units + 3) / 4 * 4;
        r.lse_floats = weights ? (B * NH + 3) / 4 * 4 : 0;
    }
    r.floats = r.part_floats + r.unit_floats + r.lse_floats + (weights ? B * NK * max_len * group : 0);
    return r;
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
    int rc = kv8_attn_check(pages, "attn_decode_q8", a.pg, block_table, bt_stride, bt_width, positions, B, 1, NH, max_len);
    if (rc != T2C_OK) return rc;
    if (!kv8_strides(q, B, q_sb, NH, q_sh, 1, 0) || !kv8_strides(out, B, o_sb, NH, o_sh, 1, 0))
        return set_error(T2C_EINVAL, "attn_decode_q8: q and out rows must be 16-byte aligned");
    if (splits < 0) return set_error(T2C_EINVAL, "attn_decode_q8: splits %lld", (long long)splits);
    const int64_t D = pages->head_dim, group = NH / a.pg.n_kv;
    if (group > 128) return set_error(T2C_EUNSUPPORTED, "attn_decode_q8: group %lld", (long long)group);
    const DecodePlan plan = decode_plan(B, NH, a.pg.n_kv, D, max_len, splits, weights_out != nullptr);
    if (plan.floats > 0 && (!workspace || workspace_floats < plan.floats))
        return set_error(T2C_ESCRATCH, "attn_decode_q8: workspace needs %lld floats", (long long)plan.floats);
    if (!kv8_aligned(workspace, 16)) return set_error(T2C_EINVAL, "attn_decode_q8: workspace must be 16-byte aligned");
    if (a.pg.n_kv * plan.head_chunks > 65535 || B * a.pg.n_kv * plan.head_chunks * ((max_len + kDTile - 1) / kDTile) > INT32_MAX)
        return set_error(T2C_EINVAL, "attn_decode_q8: bad shape");
    a.q = static_cast<const __half *>(q), a.q_sb = q_sb, a.q_sh = q_sh;
    a.out = static_cast<__half *>(out), a.o_sb = o_sb, a.o_sh = o_sh;
    a.lse = lse;
    a.positions = positions, a.table = block_table, a.t_stride = bt_stride, a.max_len = max_len;
    a.B = static_cast<int>(B), a.NH = static_cast<int>(NH);
    a.scale_log2 = scale * 1.4426950408889634f;
    const int64_t tiles = (max_len + kDTile - 1) / kDTile;
    p.splits = plan.splits, p.head_chunks = plan.head_chunks, p.ctas = plan.ctas;
    p.most_parts = static_cast<int>(p.ctas < tiles ? p.ctas : tiles);
    p.parts = workspace;
    p.unit_ctas = reinterpret_cast<int2 *>(workspace + plan.part_floats);
    p.unit_lse = workspace + plan.part_floats + plan.unit_floats;
    p.scores = workspace + plan.part_floats + plan.unit_floats + plan.lse_floats;
    p.s_len = max_len;
    p.w_in = weights, p.w_out = weights_out, p.w_sb = w_sb, p.w_sh = w_sh;
    CUtensorMap k_map, v_map;
    if (!kv8_maps(pages, 16, k_map, v_map))
        return set_error(T2C_ECUDA, "attn_decode_q8: cuTensorMapEncodeTiled failed");
    const cudaStream_t s = as_stream(stream);
    const auto kern = D == 128 ? attn8_decode_kernel<128> : attn8_decode_kernel<64>;
    const int smem = D == 128 ? DecodeShape<128>::kRing : DecodeShape<64>::kRing;
    rc = kv8_configure(kern, smem, D == 128 ? 0 : 1, "attn_decode_q8");
    if (rc != T2C_OK) return rc;
    const bool clusters = p.splits > 0;
    const dim3 grid = clusters ? dim3(static_cast<unsigned>(p.splits), static_cast<unsigned>(a.pg.n_kv * p.head_chunks),
                                      static_cast<unsigned>(B))
                               : dim3(static_cast<unsigned>(p.ctas));
    rc = kv8_launch("attn_decode_q8", kern, grid, dim3(kDThreads), smem, clusters ? static_cast<unsigned>(p.splits) : 1u, s, k_map,
                    v_map, p);
    if (rc != T2C_OK || clusters) return rc;
    // A block per head while those fit the SMs at once, then a block for as many as it has quarters (32 sequences of up to 6007,
    // 32 heads on 8: 49 us, with a block per head 54; 32801 positions of one 24, else 26).
    const int64_t chunks = weights_out ? (max_len + kJoinKeys - 1) / kJoinKeys : 0;
    const int64_t parts = p.most_parts, quarters = kJoinThreads / D;
    const bool alone = B * NH <= 4 * sm_count() || quarters * parts * 4 > 32768;
    const int64_t heads = alone ? 1 : quarters;
    const auto join = D == 128 ? (alone ? attn8_join_kernel<128, true> : attn8_join_kernel<128, false>)
                               : (alone ? attn8_join_kernel<64, true> : attn8_join_kernel<64, false>);
    return kv8_launch("attn_decode_q8 join", join,
                      dim3(static_cast<unsigned>((group + heads - 1) / heads + chunks), static_cast<unsigned>(a.pg.n_kv), static_cast<unsigned>(B)),
                      dim3(kJoinThreads), static_cast<size_t>(heads * parts * 4), 1, s, p);
}
