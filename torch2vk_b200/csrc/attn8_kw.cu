// The attention weight that many queries give each key of the paged 8-bit cache, on tcgen05.
//
// CTA = 128 keys of one (sequence, KV head), expanded to fp16 once; the query tiles that see them stream past (128 rows:
// TT = 128 / group tokens times the group's heads, fetched by TMA boxes of group x TT rows):
//   S^T = K Q^T   tcgen05.mma kind::f16, M = 128 keys, N = 128 query rows, fp32 in TMEM, two buffers
//   w_j += sum over the tile's columns of 2^(S_j kf_j - lse_col)
// Keys are the rows, so a thread owns a key: its sum needs no exchange, its K scale is a register, and the columns'
// log-sum-exps are read from shared memory by all lanes alike.  Sums are per 32 columns, per tile, then over tiles, in
// fp32 and in a fixed order.  What bounds it: the 2^ unit, one per (head, query, key); two CTAs share an SM, so that one's
// other instructions run under the other's (8192 queries of 32 heads on 8: 361 us, 0.66 of that unit's rate of 16 a clock
// and SM; with eight warps of half the columns each 369).
#include <cooperative_groups.h>
#include <cudaTypedefs.h>

#include <type_traits>

#include "kv8.cuh"
#include "umma.cuh"

namespace cg = cooperative_groups;

namespace t2c {
namespace {

constexpr int kWRows = 128;
constexpr int kWThreads = 192;  // warps 0-3: keys; 4: query tiles and log-sum-exps; 5: MMA

template <int D>
struct WeightShape {
    static constexpr int kTile = 128 * D * 2;
    static constexpr int kQ = kTile, kLse = kQ + 2 * kTile, kSums = kLse + 8 * 512, kBars = kSums + 512, kSmem = kBars + 128;
};

struct WeightArgs {
    KvPages pg;
    const float *lse;  // [B, NH, T]
    const int32_t *positions, *table;
    int64_t t_stride, max_len;
    int B, T, NH, keys_per;  // key tiles of a CTA
    float scale_log2;
    const float *w_in;
    float *w_out;
    int64_t w_sb, w_sh;
};

__device__ __forceinline__ uint32_t w_bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }

// MANY: several key tiles a CTA; without, nothing of a next tile takes registers (8192 queries of 32 heads: 361 us, else 372).
template <int D, bool MANY>
__global__ void __launch_bounds__(kWThreads, 2) attn8_weights_kernel(const __grid_constant__ CUtensorMap q_map,
                                                                     const __grid_constant__ WeightArgs a) {
    using S = WeightShape<D>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t base = smem_u32(smem);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + S::kBars);
    uint64_t *q_full = bars, *q_free = bars + 2, *s_ready = bars + 4, *s_free = bars + 6, *k_ready = bars + 8, *all_done = bars + 9;
    float *sums = reinterpret_cast<float *>(smem + S::kSums);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 10);
    volatile int *stop = reinterpret_cast<volatile int *>(bars + 11), *stop_last = stop + 1;
    if (base & 1023u) {  // the swizzle atoms need it: report, compute nothing
        if (threadIdx.x == 0) report_device_error(T2C_EUNSUPPORTED);
        return;
    }
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int group = a.NH / a.pg.n_kv, TT = kWRows / group;
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(q_full + i, 2);
            mbar_init(q_free + i, 1);
            mbar_init(s_ready + i, 1);
            mbar_init(s_free + i, 4);
        }
        mbar_init(k_ready, 4);
        mbar_init(all_done, 1);
        *stop = 0;
        fence_mbar_init();
    }
    if (TT * group < kWRows) {  // rows that no box writes
        for (int i = tid; i < 2 * S::kTile / 16; i += kWThreads)
            reinterpret_cast<uint4 *>(smem + S::kQ)[i] = make_uint4(0, 0, 0, 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 5) tmem_alloc(tmem_slot, 256);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(tmem_slot);
    pdl_wait();
    pdl_trigger();

    // blocks of the first keys, which most queries see, first; a cluster shares out the query tiles of its keys
    cg::cluster_group cluster = cg::this_cluster();
    const int C = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
    const int pairs = a.B * a.pg.n_kv, item = blockIdx.x / C;
    const int head = item % a.pg.n_kv, b = item / a.pg.n_kv % a.B;
    const int kt0 = item / pairs * (MANY ? a.keys_per : 1);
    const int64_t p0 = a.positions[b];
    int64_t n = p0 + a.T;
    if (n > a.max_len) {
        if (tid == 0) report_device_error(T2C_EINVAL);
        n = a.max_len;
    }
    const int all_keys = n > 0 ? static_cast<int>((n + 127) / 128) : 0;
    const int kt1 = min(kt0 + (MANY ? a.keys_per : 1), all_keys), nq = (a.T + TT - 1) / TT;
    // query tiles that see a key of tile kt: this CTA's share of those from the first one on
    const auto share = [&](int kt, int of) {
        const int64_t t = static_cast<int64_t>(kt) * 128 - p0;
        const int first = t <= 0 ? 0 : static_cast<int>(t / TT);
        return first + static_cast<int>(static_cast<int64_t>(nq - first) * of / C);
    };
    int loads = 0;  // query tiles that warp 4 has fetched
    if (kt0 < kt1) {
        if (warp < 4) {
            constexpr int kPerRow = D / 16, kRowsPass = 32 / kPerRow, kPasses = 32 / kRowsPass;
            const int c = D == 128 ? (lane & 3) + 4 * ((lane >> 3) & 1) : lane & 3;
            const int r0 = D == 128 ? ((lane >> 2) & 1) + 2 * (lane >> 4) : lane >> 2;
            const int32_t *bt = a.table + b * a.t_stride;
            const int page_mask = (1 << a.pg.page_log2) - 1;
            const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * warp) << 16);
            uint4 x[kPasses];
            __half ks;
            // the lane's table entry is read two tiles ahead, codes and scale one, and nothing waits for either here
            const auto entry = [&](int kt) {
                const int64_t mine = static_cast<int64_t>(kt) * 128 + 32 * warp + lane;
                return mine < n ? bt[mine >> a.pg.page_log2] : 0;
            };
            const auto fetch = [&](int kt, int page) {  // codes of the warp's 32 keys, the scale of the lane's own
                const int64_t k = static_cast<int64_t>(kt) * 128 + 32 * warp, mine = k + lane;
                if (static_cast<unsigned>(page) >= static_cast<unsigned>(a.pg.num_pages)) {
                    report_device_error(T2C_EINVAL);
                    page = 0;
                }
                ks = __ushort_as_half(0);
                if (mine < n) ks = a.pg.ks[kv8_scale_offset(a.pg, page, head, mine)];
#pragma unroll
                for (int i = 0; i < kPasses; ++i) {
                    const int r = i * kRowsPass + r0;
                    const int pg = __shfl_sync(0xffffffffu, page, r);
                    x[i] = make_uint4(0, 0, 0, 0);
                    if (k + r < n)
                        x[i] = ldg_nc_v4(a.pg.k + pg * a.pg.page_stride + head * a.pg.head_stride +
                                         (static_cast<int>(k + r) & page_mask) * a.pg.row_stride + 16 * c);
                }
            };
            const auto expand = [&]() {  // what fetch brought, as the A operand; the factor of the lane's key
#pragma unroll
                for (int i = 0; i < kPasses; ++i) {
                    const int r = 32 * warp + i * kRowsPass + r0;
                    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                    uint32_t v[8];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        __half2 even, odd;
                        kv8_unpack(w[e], even, odd);
                        v[2 * e] = __byte_perm(w_bits(even), w_bits(odd), 0x5410);
                        v[2 * e + 1] = __byte_perm(w_bits(even), w_bits(odd), 0x7632);
                    }
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const int unit = 2 * c + u;
                        const uint32_t at = base + (unit >> 3) * 16384 + r * 128 + (((unit & 7) ^ (r & 7)) << 4);
                        asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v[4 * u]), "r"(v[4 * u + 1]),
                                     "r"(v[4 * u + 2]), "r"(v[4 * u + 3])
                                     : "memory");
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(k_ready);
                return __half2float(ks) * a.scale_log2;
            };
            fetch(kt0, entry(kt0));
            int page = MANY ? entry(kt0 + 1) : 0;
            const float kf_only = MANY ? 0.0f : expand();
            int count = 0;  // query tiles so far
            for (int kt = kt0; kt < kt1; ++kt) {
                // every S of the tile before has been read, so every MMA on this buffer is done
                const float kf_tile = MANY ? expand() : kf_only;
                if (MANY && kt + 1 < kt1) fetch(kt + 1, page), page = entry(kt + 2);
                const int64_t key = static_cast<int64_t>(kt) * 128 + 32 * warp + lane;
                const uint64_t kk = f32x2(kf_tile, kf_tile);
                const int64_t o = b * a.w_sb + head * a.w_sh + key;
                const float before = C == 1 && a.w_in && key < p0 && key < n ? a.w_in[o] : 0.0f;  // on its way under the products
                float weight = 0.0f;
                for (int q = share(kt, rank), q_end = share(kt, rank + 1); q < q_end; ++q, ++count) {
                    const int buf = count & 1;
                    mbar_wait_or(&s_ready[buf], (count >> 1) & 1, stop);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t at = lanes + 128 * buf;
                    const ulonglong2 *nl = reinterpret_cast<const ulonglong2 *>(smem + S::kLse + (count & 7) * 512);
                    // columns before `from` are queries that do not see this lane's key
                    const int64_t ahead = (key - p0 - static_cast<int64_t>(q) * TT) * group;
                    const bool masked = __any_sync(0xffffffffu, ahead > 0);
                    const int from = static_cast<int>(ahead < 0 ? 0 : (ahead > 128 ? 128 : ahead));
                    // (the columns in view and the others apart: a select per column would be half of the instructions)
                    const auto columns = [&](auto hide) -> float {
                        float tile = 0.0f;
                        uint32_t s[2][32];
                        tmem_ld32(at, s[0]);
#pragma unroll
                        for (int c4 = 0; c4 < 4; ++c4) {
                            tmem_ld_wait32(s[c4 & 1]);
                            if (c4 < 3) tmem_ld32(at + 32 * (c4 + 1), s[(c4 + 1) & 1]);
                            if (c4 == 3) {  // the buffer is read
                                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                                __syncwarp();
                                if (lane == 0) mbar_arrive(&s_free[buf]);
                            }
                            uint64_t sum[2];
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const ulonglong2 two = nl[8 * c4 + (i >> 1)];
                                const uint32_t *v = s[c4 & 1] + 2 * i;
                                float2 y = f32x2_parts(f32x2_fma(f32x2(__uint_as_float(v[0]), __uint_as_float(v[1])), kk, i & 1 ? two.y : two.x));
                                if (hide) {
                                    y.x = 32 * c4 + 2 * i < from ? -INFINITY : y.x;
                                    y.y = 32 * c4 + 2 * i + 1 < from ? -INFINITY : y.y;
                                }
                                const uint64_t e = f32x2(ex2(y.x), ex2(y.y));
                                sum[i & 1] = i < 2 ? e : f32x2_add(sum[i & 1], e);
                            }
                            const float2 both = f32x2_parts(f32x2_add(sum[0], sum[1]));
                            tile += both.x + both.y;
                        }
                        return tile;
                    };
                    weight += masked ? columns(std::true_type{}) : columns(std::false_type{});
                }
                if (C > 1) {  // one key tile: the shares are summed below, in their order
                    sums[tid] = weight;
                } else if (key < n && !*stop) {
                    a.w_out[o] = weight + before;
                }
            }
        } else if (warp == 4) {
            const float *lse = a.lse + static_cast<int64_t>(b) * a.NH * a.T + static_cast<int64_t>(head) * group * a.T;
            bool on = true;
            for (int kt = kt0; kt < kt1 && on; ++kt) {
                for (int q = share(kt, rank), q_end = share(kt, rank + 1); q < q_end; ++q, ++loads) {
                    const int slot = loads & 1;
                    if (loads >= 2) on = mbar_wait_or(&q_free[slot], ((loads >> 1) - 1) & 1, stop);
                    on = __all_sync(0xffffffffu, on);
                    if (!on) break;  // no copy over one that may still be in flight
                    if (lane == 0) {
                        mbar_arrive_expect_tx(&q_full[slot], static_cast<uint32_t>(TT * group * D * 2));
#pragma unroll
                        for (int i = 0; i < D / 64; ++i)
                            tma_load_4d(base + S::kQ + slot * S::kTile + i * 16384, &q_map, 64 * i, head * group, q * TT, b, &q_full[slot]);
                    }
                    // (the ring of 8 outlives its readers) minus the log-sum-exp in log2 units; -inf (weight 0) for rows past the end and rows that see nothing
                    float *dst = reinterpret_cast<float *>(smem + S::kLse + (loads & 7) * 512);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = 32 * i + lane, t = q * TT + r / group;
                        float v = -INFINITY;
                        if (r < TT * group && t < a.T) {
                            const float x = lse[static_cast<int64_t>(r % group) * a.T + t];
                            v = x == -INFINITY ? -INFINITY : -1.4426950408889634f * x;
                        }
                        dst[r] = v;
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&q_full[slot]);
                }
            }
        } else {
            const uint32_t tm = __reduce_max_sync(0xffffffffu, tmem);
            const uint32_t idesc = umma_idesc(128, 128, false);
            int count = 0;
            for (int kt = kt0; kt < kt1; ++kt) {
                mbar_wait_or(k_ready, (kt - kt0) & 1, stop);
                for (int q = share(kt, rank), q_end = share(kt, rank + 1); q < q_end; ++q, ++count) {
                    const int slot = count & 1;
                    mbar_wait_or(&q_full[slot], (count >> 1) & 1, stop);
                    if (count >= 2) mbar_wait_or(&s_free[slot], ((count >> 1) - 1) & 1, stop);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (elect_one()) {
                        const uint32_t k = umma_desc_lo(base), qd = umma_desc_lo(base + S::kQ + slot * S::kTile);
#pragma unroll
                        for (int s = 0; s < D / 16; ++s) {
                            const uint32_t off = static_cast<uint32_t>((s >> 2) * 1024 + 2 * (s & 3));
                            umma_ss(tm + 128 * slot, k + off, qd + off, idesc, s > 0);
                        }
                        umma_commit(&s_ready[slot]);
                        umma_commit(&q_free[slot]);
                    }
                    __syncwarp();
                }
            }
            if (elect_one()) umma_commit(all_done);
            __syncwarp();
            *stop_last = 0;
            mbar_wait_or(all_done, 0, stop_last);  // nothing of this CTA is in flight when it frees its TMEM
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (*stop) {
        if (tid == 0) report_device_error(T2C_ETIMEOUT);
        if (warp == 4)  // the last copies end (or are given up) before the CTA may
            for (int i = max(loads - 2, 0); i < loads; ++i) mbar_wait(&q_full[i & 1], (i >> 1) & 1);
        __syncwarp();
    }
    if (warp == 5) {
        __syncwarp();
        tmem_free(tmem, 256);
    }
    // (TMEM is free before the wait for the cluster: its CTAs may be waiting for TMEM that other clusters' CTAs hold)
    if (C > 1) {
        cluster.sync();
        const int64_t key = static_cast<int64_t>(kt0) * 128 + tid;
        if (rank == 0 && tid < 128 && kt0 < kt1 && key < n && !*stop) {
            float weight = 0.0f;
            for (int r = 0; r < C; ++r) weight += *cluster.map_shared_rank(sums + tid, r);
            const int64_t o = b * a.w_sb + head * a.w_sh + key;
            a.w_out[o] = weight + (a.w_in && key < p0 ? a.w_in[o] : 0.0f);
        }
        cluster.sync();  // no CTA leaves while another may read its shared memory
    }
}

// Queries as (dim, head, token, sequence), boxes of 64 dims x `group` heads x `tokens`.
bool query_map(const void *q, int64_t sb, int64_t st, int64_t sh, int64_t B, int64_t T, int64_t NH, int64_t D, int group,
               int tokens, CUtensorMap &map) {
    const auto enc = kv8_encoder();
    if (!enc) return false;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(NH), static_cast<cuuint64_t>(T),
                                static_cast<cuuint64_t>(B)};
    // a dimension of one entry may have any stride: give the driver one it takes
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(NH > 1 ? sh * 2 : D * 2), static_cast<cuuint64_t>(T > 1 ? st * 2 : D * 2),
                                   static_cast<cuuint64_t>(B > 1 ? sb * 2 : D * 2)};
    const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(group), static_cast<cuuint32_t>(tokens), 1};
    const cuuint32_t es[4] = {1, 1, 1, 1};
    return enc(&map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void *>(q), dims, strides, box, es,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

cudaError_t status_attn8_kw(unsigned int *bits, int clear, cudaStream_t s) { return read_tu_status(bits, clear, s); }

}  // namespace t2c

using namespace t2c;

extern "C" int t2c_attn_key_weights_q8(const t2c_q8_pages *pages, const void *q, int64_t q_sb, int64_t q_st,
                                       int64_t q_sh, const float *lse, const int32_t *positions,
                                       const int32_t *block_table, int64_t bt_stride, int64_t bt_width, int64_t B,
                                       int64_t T, int64_t NH, float scale, int64_t max_len, const float *weights,
                                       float *weights_out, int64_t w_sb, int64_t w_sh, void *stream) {
    WeightArgs a = {};
    int rc = kv8_attn_check(pages, "attn_key_weights_q8", a.pg, block_table, bt_stride, bt_width, positions, B, T, NH, max_len);
    if (rc != T2C_OK) return rc;
    if (!kv8_strides(q, B, q_sb, T, q_st, NH, q_sh)) return set_error(T2C_EINVAL, "attn_key_weights_q8: q rows must be 16-byte aligned");
    if (!lse || !weights_out) return set_error(T2C_EINVAL, "attn_key_weights_q8: NULL pointer");
    const int64_t group = NH / a.pg.n_kv, D = pages->head_dim;
    if (group > kWRows) return set_error(T2C_EUNSUPPORTED, "attn_key_weights_q8: group %lld", (long long)group);
    const int tokens = static_cast<int>(kWRows / group);
    CUtensorMap q_map;
    if (!query_map(q, q_sb, q_st, q_sh, B, T, NH, D, static_cast<int>(group), tokens, q_map))
        return set_error(T2C_EINVAL, "attn_key_weights_q8: q's strides do not suit a tensor map");
    a.lse = lse;
    a.positions = positions, a.table = block_table, a.t_stride = bt_stride, a.max_len = max_len;
    a.B = static_cast<int>(B), a.T = static_cast<int>(T), a.NH = static_cast<int>(NH);
    a.scale_log2 = scale * 1.4426950408889634f;
    a.w_in = weights, a.w_out = weights_out, a.w_sb = w_sb, a.w_sh = w_sh;
    // Where few query tiles stream past a key tile, a CTA takes several key tiles, as many as make one wave of two CTAs per
    // SM (the next tile's codes arrive under this one).  Where many do, one, and a cluster of up to 8 CTAs shares out the
    // query tiles of the first keys, which every query sees, until the longest share is under 3/4 of the mean of an SM's
    // slot; 32 query tiles a CTA at least, which its beginning costs about 4 of (6000 queries of 16 heads on 8: 150 us
    // alone, 117 in pairs, 139 in fours; 4096 queries of 16 heads of 64 on 16: 53, 62, 84).  32 queries on 2 x 16007
    // positions: 7 key tiles a CTA 26 us, one 39.
    const int64_t nq = (T + tokens - 1) / tokens, tiles = (max_len + 127) / 128, units = B * a.pg.n_kv, slots = 2 * sm_count();
    int64_t per = nq >= 8 ? 1 : (units * tiles + slots - 1) / slots;
    per = per > 32 ? 32 : per;
    unsigned cluster = 1;
    const int64_t seen = units * (max_len > T ? (tiles - T / 128) * nq + nq * (T / 128) / 2 : nq * tiles / 2);
    while (per == 1 && cluster < 8 && nq >= 64 * cluster && (nq / cluster) * slots > seen * 3 / 4) cluster *= 2;
    a.keys_per = static_cast<int>(per);
    const int64_t blocks = units * ((tiles + per - 1) / per) * cluster;
    if (blocks > INT32_MAX) return set_error(T2C_EINVAL, "attn_key_weights_q8: bad shape");
    const auto kern = per > 1 ? (D == 128 ? attn8_weights_kernel<128, true> : attn8_weights_kernel<64, true>)
                              : (D == 128 ? attn8_weights_kernel<128, false> : attn8_weights_kernel<64, false>);
    const int smem = D == 128 ? WeightShape<128>::kSmem : WeightShape<64>::kSmem;
    rc = kv8_configure(kern, smem, (D == 128 ? 4 : 5) + (per > 1 ? 3 : 0), "attn_key_weights_q8");
    if (rc != T2C_OK) return rc;
    return kv8_launch("attn_key_weights_q8", kern, dim3(static_cast<unsigned>(blocks)), dim3(kWThreads), smem, cluster, as_stream(stream),
                      q_map, a);
}
