// Paged KV cache in 8 bits: quantized append, read back, eviction.
#include <cooperative_groups.h>
#include <math.h>

#include "kv8.cuh"

namespace cg = cooperative_groups;

namespace t2c {

int kv8_view(const t2c_q8_pages *p, const char *what, KvPages &out) {
    if (!p || !p->k || !p->v || !p->k_scale || !p->v_scale) return set_error(T2C_EINVAL, "%s: NULL pointer", what);
    const auto log2_of = [](int64_t x) {
        int l = 0;
        while ((int64_t(1) << l) < x) ++l;
        return (int64_t(1) << l) == x ? l : -1;
    };
    if (p->page_size < 16 || p->page_size > (1 << 20) || log2_of(p->page_size) < 0)
        return set_error(T2C_EINVAL, "%s: page_size %lld is not a power of two from 16 up", what, (long long)p->page_size);
    if ((p->block != 16 && p->block != 32 && p->block != 64) || p->block > p->page_size)
        return set_error(T2C_EINVAL, "%s: block %lld is not 16, 32 or 64 within a page", what, (long long)p->block);
    if (p->num_pages <= 0 || p->num_pages > INT32_MAX || p->n_kv <= 0 || p->n_kv > 65535)
        return set_error(T2C_EINVAL, "%s: bad pool shape", what);
    if (p->head_dim != 64 && p->head_dim != 128)
        return set_error(T2C_EUNSUPPORTED, "%s: head_dim %lld", what, (long long)p->head_dim);
    if (!kv8_aligned(p->k, 16) || !kv8_aligned(p->v, 16) || (p->num_pages > 1 && p->page_stride % 16) ||
        (p->n_kv > 1 && p->head_stride % 16) || p->row_stride % 16 || !kv8_aligned(p->k_scale, 2) || !kv8_aligned(p->v_scale, 2))
        return set_error(T2C_EINVAL, "%s: page rows must be 16-byte aligned", what);
    out.k = static_cast<int8_t *>(p->k);
    out.v = static_cast<int8_t *>(p->v);
    out.ks = static_cast<__half *>(p->k_scale);
    out.vs = static_cast<__half *>(p->v_scale);
    out.page_stride = p->page_stride;
    out.head_stride = p->head_stride;
    out.row_stride = p->row_stride;
    out.s_page_stride = p->scale_page_stride;
    out.s_head_stride = p->scale_head_stride;
    out.num_pages = static_cast<int>(p->num_pages);
    out.n_kv = static_cast<int>(p->n_kv);
    out.page_log2 = log2_of(p->page_size);
    out.block_log2 = log2_of(p->block);
    return T2C_OK;
}

int kv8_table(const t2c_q8_pages *p, const int32_t *table, int64_t B, int64_t stride, int64_t width, const char *what,
              int64_t &capacity) {
    if (!table) return set_error(T2C_EINVAL, "%s: NULL block table", what);
    if (width <= 0 || (B > 1 && stride < width) || width > (INT32_MAX - 65536) / p->page_size)
        return set_error(T2C_EINVAL, "%s: bad block table", what);
    capacity = width * p->page_size;
    return T2C_OK;
}

int kv8_attn_check(const t2c_q8_pages *pages, const char *what, KvPages &pg, const int32_t *table, int64_t bt_stride,
          int64_t bt_width, const int32_t *positions, int64_t B, int64_t T, int64_t NH, int64_t &max_len) {
    int64_t capacity = 0;
    int rc = kv8_view(pages, what, pg);
    if (rc == T2C_OK) rc = kv8_table(pages, table, B, bt_stride, bt_width, what, capacity);
    if (rc != T2C_OK) return rc;
    if (!positions) return set_error(T2C_EINVAL, "%s: NULL positions", what);
    if (B <= 0 || T <= 0 || NH <= 0 || NH % pg.n_kv || B > 65535 || B * T * NH > INT32_MAX)
        return set_error(T2C_EINVAL, "%s: bad shape", what);
    if (max_len <= 0 || max_len > capacity) max_len = capacity;
    return T2C_OK;
}

PFN_cuTensorMapEncodeTiled kv8_encoder() {
    static PFN_cuTensorMapEncodeTiled encode = [] {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            fn = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled>(fn);
    }();
    return encode;
}

bool kv8_maps(const t2c_q8_pages *p, int rows, CUtensorMap &k_map, CUtensorMap &v_map) {
    const auto encode = kv8_encoder();
    if (!encode) return false;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(p->head_dim), static_cast<cuuint64_t>(p->page_size),
                                static_cast<cuuint64_t>(p->n_kv), static_cast<cuuint64_t>(p->num_pages)};
    // a dimension of one entry may have any stride: give the driver one it takes
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(p->row_stride),
                                   static_cast<cuuint64_t>(p->n_kv > 1 ? p->head_stride : p->row_stride),
                                   static_cast<cuuint64_t>(p->num_pages > 1 ? p->page_stride : p->row_stride)};
    const cuuint32_t box[4] = {static_cast<cuuint32_t>(p->head_dim), static_cast<cuuint32_t>(rows), 1, 1};
    const cuuint32_t es[4] = {1, 1, 1, 1};
    const CUtensorMapSwizzle swizzle = p->head_dim == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
    CUtensorMap *maps[2] = {&k_map, &v_map};
    void *bases[2] = {p->k, p->v};
    for (int i = 0; i < 2; ++i)
        if (encode(maps[i], CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, bases[i], dims, strides, box, es,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return false;
    return true;
}

namespace {

// ------------------------------------------------------------------ write
// One CTA of four warps per (sequence, KV head, K or V, 64-row group); a warp
// owns 16 rows, so a block of 16, 32 or 64 rows is one, two or four warps.
// Rows before positions[b] in a block that gets new rows are rescaled when the
// block's scale grows; the largest new magnitude of the block crosses warps
// through shared memory.  For prompts (8191 tokens, 8 heads of 128: 50 MB in
// 13 us) a CTA's loads, barrier and stores come one after the other: DRAM is 26 %
// busy (the stores stay in the second-level cache), issue 52 %, 39 % of the warps
// are resident.  Single tokens (48 sequences: 5 us) are bound by the chain of
// position, table, scale and codes.
template <int D>
__global__ void __launch_bounds__(128) kv8_write_kernel(KvPages pg, const __half *__restrict__ k,
                                                        const __half *__restrict__ v, int64_t k_sb, int64_t k_st,
                                                        int64_t k_sh, int64_t v_sb, int64_t v_st, int64_t v_sh,
                                                        const int32_t *__restrict__ positions,
                                                        const int32_t *__restrict__ table, int64_t t_stride,
                                                        int64_t capacity, int T, int groups) {
    constexpr int kUnits = 16 * D / 8 / 32;  // 16-byte units of new rows a lane holds
    constexpr int kPerRow = D / 8;
    __shared__ uint32_t tops[4];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int group = blockIdx.x % groups;
    const int b = blockIdx.x / groups;
    const int head = blockIdx.y >> 1;
    const bool is_v = blockIdx.y & 1;
    pdl_wait();
    pdl_trigger();
    const int64_t p0 = positions[b], p1 = p0 + T;  // new rows p0 .. p1 - 1; negative ones are padding
    const int64_t slice = ((p0 > 0 ? p0 : 0) & ~int64_t(63)) + 64 * group + 16 * warp;
    const int64_t block = (slice >> pg.block_log2) << pg.block_log2;
    const int64_t block_end = block + (int64_t(1) << pg.block_log2);
    const bool touched = block < p1 && block_end > p0 && block < capacity;
    if (block >= capacity && block < p1 && block_end > p0 && lane == 0) report_device_error(T2C_EINVAL);

    const __half *src = is_v ? v + b * v_sb + head * v_sh : k + b * k_sb + head * k_sh;
    const int64_t src_t = is_v ? v_st : k_st;
    uint4 x[kUnits];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        const int u = i * 32 + lane;
        const int64_t row = slice + u / kPerRow;
        x[i] = make_uint4(0, 0, 0, 0);
        if (touched && row >= p0 && row < p1) x[i] = ldg_nc_v4(src + (row - p0) * src_t + (u % kPerRow) * 8);
        const uint32_t m = 0x7fff7fffu;
        top = __vmaxu2(top, __vmaxu2(__vmaxu2(x[i].x & m, x[i].y & m), __vmaxu2(x[i].z & m, x[i].w & m)));
    }
    top = __reduce_max_sync(0xffffffffu, max(top >> 16, top & 0xffffu));
    const int page = touched ? kv8_page(pg, table + b * t_stride, slice) : -1;
    __half *sp = (is_v ? pg.vs : pg.ks) + (page >= 0 ? kv8_scale_offset(pg, page, head, slice) : 0);
    const bool earlier = touched && block < p0;
    const float s_old = earlier && page >= 0 ? __half2float(*sp) : 0.0f;
    if (lane == 0) tops[warp] = top;
    __syncthreads();
    if (page < 0) return;
    const int per_block = 1 << (pg.block_log2 - 4);
    const int w0 = warp & ~(per_block - 1);
    for (int w = 0; w < per_block; ++w) top = max(top, tops[w0 + w]);
    // a non-finite new value (bits >= 0x7c00) or a block that already holds one: NaN
    const float s_new_rows = __half2float(
        kv8_scale_for(top >= 0x7c00u ? INFINITY : __half2float(__ushort_as_half(static_cast<unsigned short>(top)))));
    const float s = (s_new_rows != s_new_rows || s_old != s_old) ? __int_as_float(0x7fffffff) : fmaxf(s_old, s_new_rows);
    const bool ok = s > 0.0f;  // false for NaN and for an all-zero block: codes 0
    const float inv = ok ? 1.0f / s : 0.0f;
    const float2 one_over = kv8_ratio(1.0f, s, inv);
    if (lane == 0 && warp == w0) *sp = __float2half_rn(s);
    int8_t *dst = (is_v ? pg.v : pg.k) + kv8_row_offset(pg, page, head, slice);
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        const int u = i * 32 + lane;
        const int64_t row = slice + u / kPerRow;
        if (row < p0 || row >= p1) continue;
        uint64_t c[4];
        const uint32_t words[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&words[j]));
            c[j] = kv8_codes(f32x2(f.x, f.y), one_over);
        }
        uint2 out = make_uint2(kv8_pack(c[0], c[1]), kv8_pack(c[2], c[3]));
        if (!ok) out = make_uint2(0, 0);
        *reinterpret_cast<uint2 *>(dst + (row - slice) * pg.row_stride + (u % kPerRow) * 8) = out;
    }
    if (!earlier || slice >= p0 || s == s_old) return;
    // the rows already there, at the grown scale
    constexpr int kOldUnits = (16 * D / 16 + 31) / 32;
    const float2 ratio = kv8_ratio(s_old, s, inv);
#pragma unroll 1
    for (int i = 0; i < kOldUnits; ++i) {
        const int u = i * 32 + lane;
        const int64_t row = slice + u / (D / 16);
        if (row >= p0) continue;
        uint4 *at = reinterpret_cast<uint4 *>(dst + (row - slice) * pg.row_stride + (u % (D / 16)) * 16);
        uint4 codes = *at;
        uint32_t *w = reinterpret_cast<uint32_t *>(&codes);
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = ok ? kv8_recode(w[j], ratio) : 0u;
        *at = codes;
    }
}

// ------------------------------------------------------------------ read
// A thread turns 16 codes into 16 fp16 values; blockIdx.y: sequence, K or V.  (Several units a thread were slower: the
// table, scale and code loads of a unit depend on one another, and more threads hide that better.)  8191 positions of 8
// heads of 128: 50 MB in 11.5 us; 4 x 8 x 4096 rows 100 MB in 19.5 us, 5.2 TB/s.
template <int D>
__global__ void __launch_bounds__(256) kv8_read_kernel(KvPages pg, __half *__restrict__ k_out,
                                                       __half *__restrict__ v_out, const int32_t *__restrict__ first,
                                                       const int32_t *__restrict__ lengths,
                                                       const int32_t *__restrict__ table, int64_t t_stride,
                                                       int64_t capacity, int T, unsigned units) {
    constexpr unsigned kPerRow = D / 16;
    const bool is_v = blockIdx.y & 1;
    const int b = blockIdx.y >> 1;
    const unsigned per_token = static_cast<unsigned>(pg.n_kv) * kPerRow, u = blockIdx.x * 256u + threadIdx.x;
    pdl_wait();
    pdl_trigger();
    if (u >= units) return;
    const int64_t pos = static_cast<int64_t>(first[b]) + u / per_token;
    int64_t n = lengths[b];
    if (n > capacity) {
        report_device_error(T2C_EINVAL);
        n = capacity;
    }
    const int page = pos >= 0 && pos < n ? kv8_page(pg, table + b * t_stride, pos) : -1;
    uint4 out[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
    if (page >= 0) {
        const int head = static_cast<int>(u % per_token / kPerRow);
        const uint4 c = ldg_nc_v4((is_v ? pg.v : pg.k) + kv8_row_offset(pg, page, head, pos) + 16 * (u % kPerRow));
        const __half2 s = __half2half2((is_v ? pg.vs : pg.ks)[kv8_scale_offset(pg, page, head, pos)]);
        const uint32_t w[4] = {c.x, c.y, c.z, c.w};
        uint32_t *o = reinterpret_cast<uint32_t *>(out);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            __half2 even, odd;
            kv8_unpack(w[j], even, odd);
            even = __hmul2(even, s);  // exact product, rounded once
            odd = __hmul2(odd, s);
            const __half2 x = __lows2half2(even, odd), y = __highs2half2(even, odd);
            o[2 * j] = *reinterpret_cast<const uint32_t *>(&x);
            o[2 * j + 1] = *reinterpret_cast<const uint32_t *>(&y);
        }
    }
    uint4 *dst = reinterpret_cast<uint4 *>((is_v ? v_out : k_out) + static_cast<int64_t>(b) * T * pg.n_kv * D + 16ll * u);
    dst[0] = out[0];
    dst[1] = out[1];
}

// ------------------------------------------------------------------ eviction
constexpr int kEvThreads = 1024;
constexpr int kEvWarps = kEvThreads / 32;
constexpr int kEvCache = 32768;             // weights of a CTA's slice kept in shared memory
// Rows a CTA moves at a time: a warp 16 rows of K or of V.
constexpr int mv_threads(bool in_place) { return in_place ? 512 : 256; }
constexpr int mv_rows(bool in_place) { return mv_threads(in_place) / 64 * 16; }

// A weight as an integer that orders as the weights do; NaN above all, -0 as 0.
__device__ __forceinline__ uint32_t ev_key(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

__device__ __forceinline__ int ev_warp_sum(int v) { return __reduce_add_sync(0xffffffffu, v); }

// Which positions stay.  One CTA per (sequence, KV head), a cluster where the weights are more than its shared memory
// holds: the quota-th largest weight of the unprotected positions by three radix passes (11, 11, 10 bits) whose
// histograms are summed over the cluster through distributed shared memory; equal weights go to the lowest positions.
// Bound by the passes' chain of barriers: 8 us for 1003 positions, 16 us for 4 x 8 heads of 16007.
__global__ void __launch_bounds__(kEvThreads, 2) kv8_select_kernel(
    int n_kv, const float *__restrict__ weights, int64_t w_sb, int64_t w_sh, const int32_t *__restrict__ lengths, int64_t capacity,
    int cache_size, int keep, int sinks, int recent, int32_t *__restrict__ kept, int32_t *__restrict__ new_lengths) {
    extern __shared__ uint32_t cache[];
    __shared__ uint32_t hist[3][2048];
    __shared__ int warp_sure[kEvWarps], warp_eq[kEvWarps], cta_sure, cta_eq, found[2];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int head = (blockIdx.x / C) % n_kv;
    const int b = blockIdx.x / C / n_kv;
    for (int i = tid; i < 3 * 2048; i += kEvThreads) (&hist[0][0])[i] = 0;
    pdl_wait();
    pdl_trigger();
    int n = lengths[b];
    if (n > capacity || n < 0) {
        if (tid == 0) report_device_error(T2C_EINVAL);
        n = n < 0 ? 0 : static_cast<int>(capacity);
    }
    const int left = min(n, keep);
    if (rank == 0 && head == 0 && tid == 0) new_lengths[b] = left;
    const float *w = weights + b * w_sb + head * w_sh;
    int32_t *kp = kept + (static_cast<int64_t>(b) * n_kv + head) * keep;
    // this CTA's positions, and its warps' spans of them (multiples of 32 keep the order of positions)
    const int per_warp = ((n + C * kEvWarps - 1) / (C * kEvWarps) + 31) & ~31;
    const int64_t lo = static_cast<int64_t>(rank) * kEvWarps * per_warp;
    const int s0 = static_cast<int>(min(lo, static_cast<int64_t>(n)));
    const int s1 = static_cast<int>(min(lo + static_cast<int64_t>(kEvWarps) * per_warp, static_cast<int64_t>(n)));
    const bool cached = s1 - s0 <= cache_size;
    const auto key_at = [&](int pos) { return cached ? cache[pos - s0] : ev_key(w[pos]); };

    uint32_t threshold = 0xffffffffu;  // keys above it stay, and the first `ties` equal to it
    int ties = 0;
    const int mid0 = sinks, mid1 = n - recent;
    const bool choose = n > keep;
    if (choose) {
        if (cached) {
#pragma unroll 4
            for (int pos = s0 + tid; pos < s1; pos += kEvThreads) cache[pos - s0] = ev_key(w[pos]);
        }
        __syncthreads();
        int want = keep - sinks - recent;
        uint32_t prefix = 0;
        if (want > 0) {
            const int a = max(s0, mid0), z = min(s1, mid1);
            for (int pass = 0; pass < 3; ++pass) {
                const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0);
                const int bits = pass == 2 ? 10 : 11;
#pragma unroll 4
                for (int pos = a + tid; pos < z; pos += kEvThreads) {
                    const uint32_t key = key_at(pos);
                    if (pass == 0 || (key >> (shift + bits)) == prefix)
                        atomicAdd(&hist[pass][(key >> shift) & ((1u << bits) - 1)], 1u);
                }
                cluster.sync();
                // bins 2 * tid and 2 * tid + 1 over the cluster, then the bin where the count from the top reaches `want`
                int c[2] = {0, 0};
#pragma unroll 1
                for (int r0 = 0; r0 < C; r0 += 4) {  // four in flight
                    uint2 h[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        h[r] = make_uint2(0, 0);
                        if (r0 + r < C) h[r] = *reinterpret_cast<const uint2 *>(cluster.map_shared_rank(&hist[pass][2 * tid], r0 + r));
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        c[0] += static_cast<int>(h[r].x);
                        c[1] += static_cast<int>(h[r].y);
                    }
                }
                const int mine = c[0] + c[1];
                int suffix = mine;  // over this and the higher lanes
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_down_sync(0xffffffffu, suffix, o);
                    if (lane + o < 32) suffix += v;
                }
                if (lane == 0) warp_sure[warp] = suffix;
                __syncthreads();
                int above = suffix - mine;
                {
                    const int higher = lane > warp && lane < kEvWarps ? warp_sure[lane] : 0;
                    above += __reduce_add_sync(0xffffffffu, higher);
                }
                if (above < want && above + mine >= want) {
                    const bool upper = above + c[1] >= want;
                    found[0] = 2 * tid + (upper ? 1 : 0);
                    found[1] = want - above - (upper ? 0 : c[1]);
                }
                __syncthreads();
                prefix = (prefix << bits) | static_cast<uint32_t>(found[0]);
                want = found[1];
                __syncthreads();
            }
            threshold = prefix;
            ties = want;
        }
    }
    // `sure`: protected or above the threshold; `eq`: equal to it.  Counted per warp, then emitted in order.
    const int p0 = min(s0 + warp * per_warp, s1), p1 = min(p0 + per_warp, s1);
    const auto classify = [&](int pos, bool &sure, bool &eq) {
        sure = eq = false;
        if (pos >= p1) return;
        if (!choose || pos < mid0 || pos >= mid1) {
            sure = true;
        } else {
            const uint32_t key = key_at(pos);
            sure = key > threshold;
            eq = key == threshold;
        }
    };
    int n_sure = 0, n_eq = 0;
    for (int base = p0; base < p1; base += 32) {
        bool sure, eq;
        classify(base + lane, sure, eq);
        n_sure += sure;
        n_eq += eq;
    }
    n_sure = ev_warp_sum(n_sure);
    n_eq = ev_warp_sum(n_eq);
    if (lane == 0) {
        warp_sure[warp] = n_sure;
        warp_eq[warp] = n_eq;
    }
    __syncthreads();
    if (warp == 0) {
        const int a = ev_warp_sum(warp_sure[lane]), e = ev_warp_sum(warp_eq[lane]);
        if (lane == 0) cta_sure = a, cta_eq = e;
    }
    cluster.sync();
    // what comes before this warp: a lane for each lower rank and each lower warp
    int run_sure = ev_warp_sum((lane < rank ? *cluster.map_shared_rank(&cta_sure, lane) : 0) + (lane < warp ? warp_sure[lane] : 0));
    int run_eq = ev_warp_sum((lane < rank ? *cluster.map_shared_rank(&cta_eq, lane) : 0) + (lane < warp ? warp_eq[lane] : 0));
    for (int base = p0; base < p1; base += 32) {
        bool sure, eq;
        classify(base + lane, sure, eq);
        const uint32_t ms = __ballot_sync(0xffffffffu, sure), me = __ballot_sync(0xffffffffu, eq);
        const uint32_t below = (1u << lane) - 1;
        const int eq_before = run_eq + __popc(me & below);
        if (sure || (eq && eq_before < ties)) kp[run_sure + __popc(ms & below) + min(eq_before, ties)] = base + lane;
        run_sure += __popc(ms);
        run_eq += __popc(me);
    }
    for (int i = left + rank * kEvThreads + tid; i < keep; i += C * kEvThreads) kp[i] = -1;
    cluster.sync();  // no CTA leaves while another may still read its shared memory
}

// Moves the kept rows: half of a CTA's warps K, half V, in 16-row slices.  To other pages each CTA moves 64 rows.  In
// place the CTAs of a head are a cluster that walks its rows in ascending rounds of 128 a CTA, and stores once each has
// read its rows of the round: a row never moves up, so the stores of a round hit no source of a later one, and the
// next round's rows are read ahead of the stores.  (Rounds with that read-ahead, two CTAs per SM, took 41 us where CTAs of
// 64 rows take 24 when the rows go to other pages: 4 sequences of 16k positions, 4096 of 8 heads kept, 67 MB in rows of
// 128 bytes.)
template <int D, bool IN_PLACE>
__global__ void __launch_bounds__(mv_threads(IN_PLACE), IN_PLACE ? 2 : 5) kv8_move_kernel(
    KvPages pg, const float *weights, int64_t w_sb, int64_t w_sh, const int32_t *__restrict__ lengths,
    const int32_t *__restrict__ table, int64_t t_stride, int64_t capacity, const int32_t *__restrict__ out_table,
    int64_t o_stride, int keep, float *weights_out, int64_t wo_sb, int64_t wo_sh,
    const int32_t *__restrict__ kept) {
    constexpr int kWarps = mv_threads(IN_PLACE) / 32, kRowsCta = mv_rows(IN_PLACE);
    __shared__ uint32_t slice_top[2][kWarps];
    cg::cluster_group cluster = cg::this_cluster();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int chunks = gridDim.x, chunk = blockIdx.x, head = blockIdx.y, b = blockIdx.z;
    pdl_wait();
    pdl_trigger();
    const float *w = weights + b * w_sb + head * w_sh;
    float *wo = weights_out + b * wo_sb + head * wo_sh;
    int left = keep;  // to other pages the -1 of `kept` ends the rows
    const int step = chunks * kRowsCta;
    if (IN_PLACE) {
        const int n = max(min(lengths[b], static_cast<int>(min(capacity, static_cast<int64_t>(INT32_MAX)))), 0);
        if (n <= keep) {  // the whole cluster: the rows stay where they are, and so do the weights unless they have a place of their own
            if (wo != w)
                for (int i = chunk * blockDim.x + threadIdx.x; i < n; i += chunks * blockDim.x) wo[i] = w[i];
            return;
        }
    }
    const int32_t *bt = table + b * t_stride, *bo = out_table + b * o_stride;
    const int32_t *kp = kept + (static_cast<int64_t>(b) * pg.n_kv + head) * keep;
    const bool is_v = warp >= kWarps / 2;
    const int slice_of = warp & (kWarps / 2 - 1);
    int8_t *codes = is_v ? pg.v : pg.k;
    __half *scales = is_v ? pg.vs : pg.ks;
    constexpr int kUnits = D / 64 * 2;  // 16-byte units of 16 rows per lane
    constexpr int kPerRow = D / 16;

    uint4 x[kUnits];
    float s_src = 0.0f, w_val = 0.0f;  // of row lane & 15 of the slice
    int rows = 0;                      // of the slice
    const auto fetch = [&](int r0) {
        const int row0 = r0 + chunk * kRowsCta + 16 * slice_of, my_row = row0 + (lane & 15);
        int64_t src = 0;
        s_src = 0.0f;
        const int pos = my_row < left ? kp[my_row] : -1;
        rows = __popc(__ballot_sync(0xffffffffu, lane < 16 && pos >= 0));
        if (pos >= 0) {
            const int page = max(kv8_page(pg, bt, pos), 0);
            src = kv8_row_offset(pg, page, head, pos);
            s_src = __half2float(scales[kv8_scale_offset(pg, page, head, pos)]);
            if (!is_v) w_val = w[pos];
        }
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const int u = i * 32 + lane, row = u / kPerRow;
            const int64_t at = __shfl_sync(0xffffffffu, src, row);
            x[i] = make_uint4(0, 0, 0, 0);
            if (row < rows) x[i] = *reinterpret_cast<const uint4 *>(codes + at + (u % kPerRow) * 16);
        }
    };
    fetch(0);
    for (int r0 = 0, round = 0; r0 < (IN_PLACE ? left : 1); r0 += step, ++round) {
        const int row0 = r0 + chunk * kRowsCta + 16 * slice_of, my_row = row0 + (lane & 15);
        float top = 0.0f;
        uint4 q[kUnits];
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const float s_row = __shfl_sync(0xffffffffu, s_src, (i * 32 + lane) / kPerRow);
            q[i] = x[i];
            uint32_t most = 0, least = 0;
            kv8_extremes(q[i].x, most, least);
            kv8_extremes(q[i].y, most, least);
            kv8_extremes(q[i].z, most, least);
            kv8_extremes(q[i].w, most, least);
            top = s_row != s_row ? INFINITY : fmaxf(top, static_cast<float>(kv8_largest(most, least)) * s_row);
        }
        const float w_row = w_val, s_mine = s_src;
        const int mine = rows;
        const uint32_t top_bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
        uint32_t *tops = slice_top[round & 1];
        if (lane == 0) tops[warp] = top_bits;
        if (IN_PLACE) {
            cluster.sync();
            if (r0 + step < left) fetch(r0 + step);
        } else {
            __syncthreads();
        }
        const int per_block = 1 << (pg.block_log2 - 4);
        const int w0 = warp & ~(per_block - 1);
        uint32_t best = 0;
        for (int i = 0; i < per_block; ++i) best = max(best, tops[w0 + i]);
        const __half s_half = kv8_scale_for(__uint_as_float(best));
        const float s = __half2float(s_half);
        const bool ok = s > 0.0f;
        const float inv = ok ? 1.0f / s : 0.0f;
        if (mine == 0) continue;
        const int page = kv8_page(pg, bo, row0);
        if (page < 0) continue;
        if (lane == 0 && warp == w0) scales[kv8_scale_offset(pg, page, head, row0)] = s_half;
        int8_t *dst = codes + kv8_row_offset(pg, page, head, row0) + lane / kPerRow * pg.row_stride + lane % kPerRow * 16;
        const float2 own = kv8_ratio(s_mine, s, inv);
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const int row = (i * 32 + lane) / kPerRow;
            const float2 ratio = make_float2(__shfl_sync(0xffffffffu, own.x, row), __shfl_sync(0xffffffffu, own.y, row));
            uint4 v = make_uint4(0, 0, 0, 0);
            if (ok) v = make_uint4(kv8_recode(q[i].x, ratio), kv8_recode(q[i].y, ratio), kv8_recode(q[i].z, ratio), kv8_recode(q[i].w, ratio));
            if (row < mine) *reinterpret_cast<uint4 *>(dst + i * (32 / kPerRow) * pg.row_stride) = v;
        }
        if (!is_v && lane < mine) wo[my_row] = w_row;
    }
}

}  // namespace

cudaError_t status_kv8(unsigned int *bits, int clear, cudaStream_t s) { return read_tu_status(bits, clear, s); }

}  // namespace t2c

using namespace t2c;

extern "C" int t2c_kv_cache_write_q8(const t2c_q8_pages *pages, const void *k, int64_t k_sb, int64_t k_st, int64_t k_sh,
                                     const void *v, int64_t v_sb, int64_t v_st, int64_t v_sh, const int32_t *positions,
                                     const int32_t *block_table, int64_t bt_stride, int64_t bt_width, int64_t B,
                                     int64_t T, void *stream) {
    KvPages pg;
    int64_t capacity = 0;
    int rc = kv8_view(pages, "kv_cache_write_q8", pg);
    if (rc == T2C_OK) rc = kv8_table(pages, block_table, B, bt_stride, bt_width, "kv_cache_write_q8", capacity);
    if (rc != T2C_OK) return rc;
    if (!k || !v || !positions) return set_error(T2C_EINVAL, "kv_cache_write_q8: NULL pointer");
    if (B <= 0 || T <= 0 || T > INT32_MAX - 128) return set_error(T2C_EINVAL, "kv_cache_write_q8: bad shape");
    if (!kv8_strides(k, B, k_sb, T, k_st, pg.n_kv, k_sh) || !kv8_strides(v, B, v_sb, T, v_st, pg.n_kv, v_sh))
        return set_error(T2C_EINVAL, "kv_cache_write_q8: rows must be 16-byte aligned");
    const int64_t groups = (T + 62) / 64 + 1;  // 64-row groups that T rows from any position can touch
    if (B * groups > INT32_MAX || pg.n_kv > 32767) return set_error(T2C_EINVAL, "kv_cache_write_q8: bad shape");
    const auto kern = pages->head_dim == 128 ? kv8_write_kernel<128> : kv8_write_kernel<64>;
    return kv8_launch("kv_cache_write_q8", kern, dim3(static_cast<unsigned>(B * groups), static_cast<unsigned>(2 * pg.n_kv)),
                      dim3(128), 0, 1, as_stream(stream), pg, static_cast<const __half *>(k),
                      static_cast<const __half *>(v), k_sb, k_st, k_sh, v_sb, v_st, v_sh, positions, block_table, bt_stride,
                      capacity, static_cast<int>(T), static_cast<int>(groups));
}

extern "C" int t2c_kv_cache_read_q8(const t2c_q8_pages *pages, void *k_out, void *v_out, const int32_t *first,
                                    const int32_t *lengths, const int32_t *block_table, int64_t bt_stride,
                                    int64_t bt_width, int64_t B, int64_t T, void *stream) {
    KvPages pg;
    int64_t capacity = 0;
    int rc = kv8_view(pages, "kv_cache_read_q8", pg);
    if (rc == T2C_OK) rc = kv8_table(pages, block_table, B, bt_stride, bt_width, "kv_cache_read_q8", capacity);
    if (rc != T2C_OK) return rc;
    if (!k_out || !v_out || !first || !lengths) return set_error(T2C_EINVAL, "kv_cache_read_q8: NULL pointer");
    if (B <= 0 || T <= 0 || T > INT32_MAX) return set_error(T2C_EINVAL, "kv_cache_read_q8: bad shape");
    if (!kv8_aligned(k_out, 16) || !kv8_aligned(v_out, 16))
        return set_error(T2C_EINVAL, "kv_cache_read_q8: outputs must be 16-byte aligned");
    const int64_t units = T * pg.n_kv * (pages->head_dim / 16);  // of a sequence
    if (units > INT32_MAX - 1024 || B > 32767) return set_error(T2C_EINVAL, "kv_cache_read_q8: bad shape");
    const int64_t blocks = (units + 255) / 256;
    const auto kern = pages->head_dim == 128 ? kv8_read_kernel<128> : kv8_read_kernel<64>;
    return kv8_launch("kv_cache_read_q8", kern, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(2 * B)),
                      dim3(256), 0, 1, as_stream(stream), pg,
                      static_cast<__half *>(k_out), static_cast<__half *>(v_out), first, lengths, block_table, bt_stride,
                      capacity, static_cast<int>(T), static_cast<unsigned>(units));
}

extern "C" int t2c_kv_cache_evict_q8(const t2c_q8_pages *pages, const float *weights, int64_t w_sb, int64_t w_sh,
                                     const int32_t *lengths, const int32_t *block_table, int64_t bt_stride,
                                     int64_t bt_width, const int32_t *out_table, int64_t ot_stride, int64_t ot_width,
                                     int64_t B, int64_t keep, int64_t sinks, int64_t recent, float *weights_out,
                                     int64_t wo_sb, int64_t wo_sh, int32_t *kept, int32_t *new_lengths, void *stream) {
    KvPages pg;
    int64_t capacity = 0, out_capacity = 0;
    int rc = kv8_view(pages, "kv_cache_evict_q8", pg);
    if (rc == T2C_OK) rc = kv8_table(pages, block_table, B, bt_stride, bt_width, "kv_cache_evict_q8", capacity);
    if (rc == T2C_OK) rc = kv8_table(pages, out_table, B, ot_stride, ot_width, "kv_cache_evict_q8", out_capacity);
    if (rc != T2C_OK) return rc;
    if (B <= 0) return set_error(T2C_EINVAL, "kv_cache_evict_q8: bad shape");
    if (sinks < 0 || recent < 0 || keep <= 0 || sinks + recent > keep)
        return set_error(T2C_EINVAL, "kv_cache_evict_q8: needs keep > 0, sinks >= 0, recent >= 0 and sinks + recent <= keep");
    if (!weights || !lengths || !weights_out || !kept || !new_lengths)
        return set_error(T2C_EINVAL, "kv_cache_evict_q8: NULL pointer");
    if (lengths == new_lengths) return set_error(T2C_EINVAL, "kv_cache_evict_q8: new_lengths must not be lengths");
    if (keep > out_capacity)
        return set_error(T2C_EINVAL, "kv_cache_evict_q8: keep %lld exceeds the %lld positions of out_table", (long long)keep,
                         (long long)out_capacity);
    const bool in_place = out_table == block_table;
    if (in_place && B > 1 && ot_stride != bt_stride) return set_error(T2C_EINVAL, "kv_cache_evict_q8: one table with two strides");
    if (!in_place && weights == weights_out)
        return set_error(T2C_EINVAL, "kv_cache_evict_q8: weights in place need the codes in place");
    if (weights == weights_out && ((B > 1 && w_sb != wo_sb) || (pg.n_kv > 1 && w_sh != wo_sh)))
        return set_error(T2C_EINVAL, "kv_cache_evict_q8: one tensor of weights with two strides");
    const int64_t heads = B * pg.n_kv;
    // CTAs that select for a head: up to 8 while the SMs have room and each keeps 2048 positions (select, move and read back,
    // 8 heads: 16007 positions of 4 sequences 55 us, one CTA a head 62, eight 70; 60000 of one 70, one CTA 160; 1003 of one
    // 13, eight 20)
    unsigned cluster = 1;
    while (cluster < 8 && capacity > static_cast<int64_t>(cluster) * 4096 &&
           (heads * cluster * 2 <= sm_count() || capacity > static_cast<int64_t>(cluster) * kEvCache))
        cluster *= 2;
    const int64_t slice = (capacity + cluster - 1) / cluster + 32 * kEvWarps;
    const int cache = static_cast<int>(slice < kEvCache ? slice : kEvCache);
    int64_t chunks = (keep + mv_rows(in_place) - 1) / mv_rows(in_place);
    if (in_place) {  // a cluster per head, as large as gives every SM a CTA, up to 8 (4096 of 16384 positions, 4 sequences of 8
                     // heads: 38 us, one CTA a head 175; 1024 of 2048, 32 sequences: one 57, two 60, eight 63)
        const int64_t full = chunks;
        chunks = 1;
        while (chunks < 8 && chunks < full && heads * chunks < sm_count()) chunks *= 2;
    }
    if (heads * cluster > INT32_MAX || B > 65535) return set_error(T2C_EINVAL, "kv_cache_evict_q8: bad shape");
    rc = kv8_configure(kv8_select_kernel, kEvCache * 4, 6, "kv_cache_evict_q8");
    // not resident early: CTAs of 1024 threads in wait slowed the kernel before them (4096 of 16384 positions of 4 sequences in
    // place, call after call: 38 us, with early residence 48)
    if (rc == T2C_OK)
        rc = kv8_launch_as(false, "kv_cache_evict_q8", kv8_select_kernel, dim3(static_cast<unsigned>(heads * cluster)), dim3(kEvThreads),
                        static_cast<size_t>(cache) * 4, cluster, as_stream(stream), pg.n_kv, weights, w_sb, w_sh, lengths, capacity, cache,
                        static_cast<int>(keep), static_cast<int>(sinks), static_cast<int>(recent), kept, new_lengths);
    if (rc != T2C_OK) return rc;
    const bool wide = pages->head_dim == 128;
    const auto kern = in_place ? (wide ? kv8_move_kernel<128, true> : kv8_move_kernel<64, true>)
                               : (wide ? kv8_move_kernel<128, false> : kv8_move_kernel<64, false>);
    return kv8_launch("kv_cache_evict_q8 move", kern,
                      dim3(static_cast<unsigned>(chunks), static_cast<unsigned>(pg.n_kv), static_cast<unsigned>(B)), dim3(mv_threads(in_place)), 0,
                      in_place ? static_cast<unsigned>(chunks) : 1u, as_stream(stream), pg, weights, w_sb, w_sh, lengths,
                      block_table, bt_stride, capacity, out_table, ot_stride, static_cast<int>(keep),
                      weights_out, wo_sb, wo_sh, kept);
}
