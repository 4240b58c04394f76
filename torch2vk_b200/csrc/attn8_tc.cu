// Attention of many query tokens over the paged 8-bit KV cache on tcgen05.
//
// CTA = two query tiles of one (sequence, KV head) and a run of its key tiles.  A query tile is 128 rows: TT =
// 128 / group tokens times the group's heads, so that one expansion of a key tile serves the whole group; row r is
// token r / group, head r % group, and TMEM lane r.  Per 128-key tile j and query tile i:
//   S_i = Q_i K_j^T     tcgen05.mma kind::f16, M = 128 rows, N = 128 keys, K = D, fp32 in TMEM
//   P_i = 2^(S_i kf_j + log2 vs_j - m)   fp16 over S_i's columns in TMEM (A operand of the next product)
//   O_i += P_i V_j      N = D, K = 128 keys, V as an MN-major operand
// Roles: warps 0-3 and 4-7 the softmax of the two query tiles (a thread one row), warps 8-15 expand the int8 codes
// to fp16 operand tiles (loads a tile ahead in registers), warp 16 issues the MMAs.
//
// The tensor core's work for one query tile runs under the other tile's softmax.  What bounds it: the chain S, softmax, P V
// of a query tile, whose P takes the place of its S (TMEM holds two S and two O of 128 columns, no third S).  With D = 64 a
// third S fits: the three go round, S of the next key tile is made while this one's softmax runs, and the chain is the
// softmax alone (4 x 512 queries on up to 3500, 16 heads of 64 on 16: 65 us, with two 73).  8192 queries
// on themselves, 32 heads of 128 on 8: 582 us, 945 TFLOP/s; a key tile takes 3800 clocks, of them the softmax 2150 (the 2^
// unit 1024), the products 1010, two hand-overs through mbarriers 550, where the products alone would take 2020 and the 2^
// of both query tiles 2050.  Measured and not kept: four softmax warpgroups, half a row a thread (643 us), S in halves of
// 64 keys (607), P handed over in halves (660), 16 keys a stage (690), one lane polling the barriers (875).
//
// Codes become fp16 exactly.  The scales stay in fp32 in the exponent: kf = k scale * softmax scale * log2 e; the V
// scale joins as log2 vs, and the softmax sum takes P / vs.  One reference m per row serves all tiles until the P of
// 16 keys sum to more than 2^14: then the row's m moves to those keys' maximum - 8 (a whole number, so that rescaling
// by 2^(old - new) is exact) and O, l and the tile's P are rescaled.  So no pass looks for the maximum; P's rounding
// to fp16 (what the tensor core takes) is the only one before the output's, but for P that a move brings below fp16's
// normal numbers: those round once more, by at most 2^-25 where the row's largest P is 2^8 or more.
//
// Within groups of four dims K and Q rows are held in the order 0, 2, 1, 3 (as the expansion leaves them; the product
// does not see it), V's columns too, which the epilogue undoes.
#include <type_traits>

#include "kv8.cuh"
#include "umma.cuh"

namespace t2c {
namespace {

constexpr int kPRows = 128;   // rows of a query tile
constexpr int kPKeys = 128;   // keys of a tile
constexpr int kPThreads = 640;
constexpr float kPRefStart = -1e30f;
constexpr float kPSumTop = 16384.0f;  // sum of 16 P that moves the reference; 16 P of 2^10 do not
constexpr float kPRefMove = 10.0f;
constexpr float kPRefDrop = 8.0f;

template <int D>
struct PrefillShape {
    static constexpr int kTile = 128 * D * 2;          // bytes of a 128-row fp16 tile: D / 64 chunks of 16 KB
    static constexpr int kQ = 0, kK = 2 * kTile, kV = kK + 2 * kTile, kMeta = kV + 2 * kTile;
    static constexpr int kBars = kMeta + 4 * 8 * 20;   // meta: ring of 4 tiles x 8 groups of 16 keys
    static constexpr int kSmem = kBars + 256;
    static constexpr int kS = D == 64 ? 3 : 2;         // S buffers of 128 TMEM columns that lie beside the two O
    static constexpr int kO = 128 * kS;
};

struct PrefillArgs {
    KvPages pg;
    const __half *q;
    int64_t q_sb, q_st, q_sh;
    __half *out;
    int64_t o_sb, o_st, o_sh;
    float *lse;
    const int32_t *positions, *table;
    int64_t t_stride, max_len;
    int B, T, NH, pairs, splits;
    float scale_log2;
    float *parts;  // [B][n_kv][pairs][splits][256][D + 2]: O rows, then m and l of 256 rows
};

__device__ __forceinline__ uint32_t ph_bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }

// byte offset of 16-byte unit u of row r of a tile: 64-value chunks of 16 KB, 128-byte swizzle
__device__ __forceinline__ uint32_t unit_at(int r, int u) {
    return static_cast<uint32_t>((u >> 3) * 16384 + r * 128 + (((u & 7) ^ (r & 7)) << 4));
}

__device__ __forceinline__ void sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// Registers of the roles, of the 640 x 96 the CTA has: 2 x 136 + 2 x 72 + 64 = 5 x 96.
template <int R>
__device__ __forceinline__ void more_registers() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R));
}
template <int R>
__device__ __forceinline__ void fewer_registers() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R));
}

template <int D>
__global__ void __launch_bounds__(kPThreads, 1) attn8_prefill_kernel(const __grid_constant__ PrefillArgs a) {
    using S = PrefillShape<D>;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t base = smem_u32(smem);
    // per group of 16 keys: (K factor twice, log2 V scale twice), and 1 / V scale
    ulonglong2 *meta = reinterpret_cast<ulonglong2 *>(smem + S::kMeta);
    float *inv_vs = reinterpret_cast<float *>(smem + S::kMeta + 4 * 8 * 16);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + S::kBars);
    uint64_t *k_full = bars, *v_full = bars + 2, *k_free = bars + 4, *v_free = bars + 6, *o_added = bars + 8, *o_done = bars + 10,
             *s_ready = bars + 11, *p_ready = bars + 14, *q_full = bars + 17, *meta_full = bars + 18;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 22);
    volatile int *stop = reinterpret_cast<volatile int *>(bars + 23), *stop_last = stop + 1;
    int *nan_from = reinterpret_cast<int *>(bars + 24);  // first key of this CTA's tiles whose V reads as NaN
    if (base & 1023u) {  // the swizzle atoms need it: report, compute nothing
        if (threadIdx.x == 0) report_device_error(T2C_EUNSUPPORTED);
        return;
    }
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        for (int i = 0; i < 4; ++i) mbar_init(k_full + i, 8);  // k_full, v_full: the expanding warps
        for (int i = 4; i < 14; ++i) mbar_init(bars + i, 1);   // commits
        for (int i = 0; i < 3; ++i) mbar_init(p_ready + i, 4);
        mbar_init(q_full, 256);
        for (int i = 0; i < 4; ++i) mbar_init(meta_full + i, 8);
        *stop = 0;
        *nan_from = INT32_MAX;
        fence_mbar_init();
    }
    if (warp == 16) tmem_alloc(tmem_slot, 512);
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(tmem_slot);
    pdl_wait();
    pdl_trigger();

    // ---- this CTA's item: the pairs with most keys first
    const int group = a.NH / a.pg.n_kv, TT = kPRows / group;
    int item = blockIdx.x;
    const int split = item % a.splits;
    item /= a.splits;
    const int head = item % a.pg.n_kv;
    item /= a.pg.n_kv;
    const int b = item % a.B;
    const int pair = a.pairs - 1 - item / a.B;
    const int t_first = pair * 2 * TT, t_last = min(t_first + 2 * TT, a.T) - 1;
    if (warp < 8) {  // a warp 32 rows of a query tile, neighbouring lanes neighbouring units of a row, all loads in flight (sixteen
        // of D = 128: the row tiles are there 0.7 us earlier than in two turns of eight), before positions are known
        const int qi = warp >> 2;
        constexpr int kUnits = D / 8, kRowsPer = 32 / kUnits, kLoads = 32 / kRowsPer;
        const uint32_t at = base + S::kQ + qi * S::kTile;
        const int u = lane % kUnits, r0 = 32 * (warp & 3) + lane / kUnits;
        const uint32_t per = 65536u / group + 1;  // r / group = r * per >> 16 for r, group <= 128
        const __half *src = a.q + b * a.q_sb + static_cast<int64_t>(head * group) * a.q_sh + 8 * u;
        uint4 v[kLoads];
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int r = r0 + i * kRowsPer, tr = r * per >> 16, tq = t_first + qi * TT + tr;
            v[i] = make_uint4(0, 0, 0, 0);
            if (tr < TT && tq < a.T)
                v[i] = *reinterpret_cast<const uint4 *>(src + static_cast<int64_t>(tq) * a.q_st + (r - tr * group) * a.q_sh);
        }
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
            sts128(at + unit_at(r0 + i * kRowsPer, u), __byte_perm(v[i].x, v[i].y, 0x5410), __byte_perm(v[i].x, v[i].y, 0x7632),
                   __byte_perm(v[i].z, v[i].w, 0x5410), __byte_perm(v[i].z, v[i].w, 0x7632));
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(q_full);
    }
    const int64_t p0 = a.positions[b];
    int64_t n = p0 + t_last + 1;  // keys the last query sees
    if (n > a.max_len) {
        if (tid == 0) report_device_error(T2C_EINVAL);
        n = a.max_len;
    }
    if (n < 0) n = 0;
    const int all_tiles = static_cast<int>((n + kPKeys - 1) / kPKeys);
    const int per = (all_tiles + a.splits - 1) / a.splits;
    const int tile0 = min(split * per, all_tiles), tiles = min(per, all_tiles - tile0);

    if (tiles > 0) {
        if (warp < 8) {
            // ================================================== softmax: tile `qi`, row `row`
            more_registers<136>();
            const int qi = warp >> 2, row = tid & 127;
            const int t = t_first + qi * TT + row / group, h = head * group + row % group;
            const bool real = row < TT * group && t < a.T;
            // last key of this row, and of the tile's first token: rows past the end follow the last real token
            const int64_t limit = min(p0 + min(t, a.T - 1), n - 1);
            const int64_t least = min(p0 + min(t_first + qi * TT, a.T - 1), n - 1);
            const uint32_t lanes = tmem + (static_cast<uint32_t>(32 * (warp & 3)) << 16);
            const uint32_t o_at = lanes + S::kO + D * qi;
            float m = kPRefStart, l = 0.0f;
            // S of (key tile j, query tile qi) is number 2 j + qi, in buffer number % kS
            int buf = qi, turn = 0;
            for (int j = 0; j < tiles; ++j, buf += 2 - S::kS, turn ^= 1) {
                if (buf < 0) buf += S::kS, turn ^= 1;  // (two numbers on wrap round or not)
                const uint32_t s_at = lanes + 128 * buf;
                mbar_wait_or(&meta_full[j & 3], (j >> 2) & 1, stop);
                const ulonglong2 *f = meta + (j & 3) * 8;
                const float *fi = inv_vs + (j & 3) * 8;
                // the factors come to registers before S is there: shared memory is slow to answer under the MMAs' reads
                float kf[8], lv[8], iv[8];
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const float4 x = reinterpret_cast<const float4 *>(f)[c];
                    kf[c] = x.x, lv[c] = x.z, iv[c] = fi[c];
                }
                mbar_wait_or(&s_ready[buf], turn, stop);
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const int64_t k0 = static_cast<int64_t>(tile0 + j) * kPKeys;
                const bool masked = k0 + kPKeys - 1 > least;

                // 32 keys at a time, three stages deep: exponents of chunk r (its S loaded before), 2^, sums and fp16 of
                // chunk r - 1, check and store of chunk r - 2.  P of chunk c goes over S columns 16 c .. 16 c + 15, all
                // read by then.  Returns the group of 16 keys from which another reference is needed, or 8.
                const int last = static_cast<int>(max(min(limit - k0, static_cast<int64_t>(kPKeys)), static_cast<int64_t>(-1)));
                const auto fast = [&](auto hide) -> int {
                    uint32_t s[32], p[2][16];
                    uint64_t y[2][16];
                    float total[2][2];
                    tmem_ld32(s_at, s);
#pragma unroll
                    for (int r = 0; r < 6; ++r) {
                        if (r >= 2) {
                            const int c = r - 2;
                            if (__any_sync(0xffffffffu, fmaxf(total[c & 1][0], total[c & 1][1]) > kPSumTop)) {
                                tmem_ld_wait();  // the load ahead
                                return 2 * c;
                            }
                            l = fmaf(total[c & 1][0], iv[2 * c], l);
                            l = fmaf(total[c & 1][1], iv[2 * c + 1], l);
                            tmem_st16(s_at + 16 * c, p[c & 1]);
                        }
                        if (r < 4) {
                            tmem_ld_wait32(s);
                            const uint64_t k0 = f32x2(kf[2 * r], kf[2 * r]), k1 = f32x2(kf[2 * r + 1], kf[2 * r + 1]);
                            const float h0 = lv[2 * r] - m, h1 = lv[2 * r + 1] - m;
                            const uint64_t shift0 = f32x2(h0, h0), shift1 = f32x2(h1, h1);
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                y[r & 1][i] = f32x2_fma(f32x2(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), i < 8 ? k0 : k1,
                                                   i < 8 ? shift0 : shift1);
                                if (hide) {
                                    const float2 v = f32x2_parts(y[r & 1][i]);
                                    y[r & 1][i] = f32x2(32 * r + 2 * i > last ? -INFINITY : v.x, 32 * r + 2 * i + 1 > last ? -INFINITY : v.y);
                                }
                            }
                            if (r < 3) tmem_ld32(s_at + 32 * (r + 1), s);
                        }
                        if (r >= 1 && r < 5) {
                            const int c = (r - 1) & 1;
                            uint64_t sum[4];
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const float2 v = f32x2_parts(y[c][i]);
                                const float e0 = ex2(v.x), e1 = ex2(v.y);
                                const int k = (i >> 3) * 2 + (i & 1);
                                sum[k] = (i & 7) < 2 ? f32x2(e0, e1) : f32x2_add(sum[k], f32x2(e0, e1));
                                p[c][i] = ph_bits(__floats2half2_rn(e0, e1));
                            }
                            const float2 t0 = f32x2_parts(f32x2_add(sum[0], sum[1])), t1 = f32x2_parts(f32x2_add(sum[2], sum[3]));
                            total[c][0] = t0.x + t0.y;
                            total[c][1] = t1.x + t1.y;
                        }
                    }
                    return 8;
                };
                // Moves the reference of the rows that need it to the maximum of groups c0 .. 7, a whole number - 8 on; O, l and
                // the P of this tile so far are rescaled.  In the first tile of a CTA, and rarely after it.
                const auto move_reference = [&](int c0) {
                    float top = -INFINITY;
#pragma unroll 1
                    for (int c = c0; c < 8; ++c) {
                        uint32_t v[16];
                        tmem_ld16(s_at + 16 * c, v);
                        const float kf = f32x2_parts(f[c].x).x, lv = f32x2_parts(f[c].y).x;
                        tmem_ld_wait16(v);
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float x = fmaf(__uint_as_float(v[i]), kf, lv);
                            top = fmaxf(top, 16 * c + i > last ? -INFINITY : x);
                        }
                    }
                    const float ref = top - m > kPRefMove ? floorf(top) - kPRefDrop : m;
                    const float corr = ex2(m - ref);
                    m = ref;
                    l *= corr;
                    if (j > 0) {
                        if (S::kS > 2) {  // (with two buffers S being ready says that the tiles before are in O)
                            mbar_wait_or(&o_added[qi], (j - 1) & 1, stop);
                            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        }
#pragma unroll 1
                        for (int i = 0; i < D / 16; ++i) {
                            uint32_t w[16];
                            tmem_ld16(o_at + 16 * i, w);
                            tmem_ld_wait16(w);
#pragma unroll
                            for (int k = 0; k < 16; ++k) w[k] = __float_as_uint(__uint_as_float(w[k]) * corr);
                            tmem_st16(o_at + 16 * i, w);
                        }
                    }
                    if (c0 > 0) tmem_st_wait();  // P is read back
#pragma unroll 1
                    for (int i = 0; i < c0; ++i) {
                        uint32_t w[8];
                        tmem_ld8(s_at + 8 * i, w);
                        tmem_ld_wait8(w);
#pragma unroll
                        for (int k = 0; k < 8; ++k) {  // in fp32: corr may be below fp16's least number
                            const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&w[k]));
                            w[k] = ph_bits(__floats2half2_rn(x.x * corr, x.y * corr));
                        }
                        tmem_st8(s_at + 8 * i, w);
                    }
                };
                // Groups c0 .. 7 after the reference moved.
                const auto rest = [&](int c0) {
#pragma unroll 1
                    for (int c = c0; c < 8; ++c) {
                        uint32_t v[16], p[8];
                        tmem_ld16(s_at + 16 * c, v);
                        const float kf = f32x2_parts(f[c].x).x, shift = f32x2_parts(f[c].y).x - m;
                        tmem_ld_wait16(v);
                        float sum = 0.0f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            float a0 = ex2(fmaf(__uint_as_float(v[2 * i]), kf, shift)), a1 = ex2(fmaf(__uint_as_float(v[2 * i + 1]), kf, shift));
                            a0 = 16 * c + 2 * i > last ? 0.0f : a0;
                            a1 = 16 * c + 2 * i + 1 > last ? 0.0f : a1;
                            sum += a0 + a1;
                            p[i] = ph_bits(__floats2half2_rn(a0, a1));
                        }
                        l = fmaf(sum, fi[c], l);
                        tmem_st8(s_at + 8 * c, p);
                    }
                };
                if (j == 0) move_reference(0);
                const int done = masked ? fast(std::true_type{}) : fast(std::false_type{});
                if (done < 8) {
                    move_reference(done);
                    rest(done);
                }
                tmem_st_wait();
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_ready[buf]);
            }
            mbar_wait_or(o_done, 0, stop);
            if (!__any_sync(0xffffffffu, *stop != 0)) {
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const bool seen = limit >= 0, poisoned = limit >= *nan_from;  // (written before the factors of those keys)
                if (a.splits > 1) {
                    float *part = a.parts + (((static_cast<int64_t>(b) * a.pg.n_kv + head) * a.pairs + pair) * a.splits + split) *
                                                (256 * (D + 2));
                    float *dst = part + (qi * 128 + row) * D;
#pragma unroll 1
                    for (int c = 0; c < D / 32; ++c) {
                        uint32_t v[32];
                        tmem_ld32(o_at + 32 * c, v);
                        tmem_ld_wait32(v);
                        if (poisoned) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = 0x7fffffffu;
                        }
                        if (real) {
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                reinterpret_cast<uint4 *>(dst)[8 * c + i] = make_uint4(v[4 * i], v[4 * i + 2], v[4 * i + 1], v[4 * i + 3]);
                        }
                    }
                    part[256 * D + qi * 128 + row] = m;
                    part[256 * (D + 1) + qi * 128 + row] = l;
                } else {
                    const float inv = poisoned ? __int_as_float(0x7fffffff) : (seen ? 1.0f / l : 0.0f);
                    __half *o = a.out + b * a.o_sb + static_cast<int64_t>(t) * a.o_st + h * a.o_sh;
#pragma unroll 1
                    for (int c = 0; c < D / 32; ++c) {
                        uint32_t v[32];
                        tmem_ld32(o_at + 32 * c, v);
                        tmem_ld_wait32(v);
                        float x[32];
#pragma unroll
                        for (int i = 0; i < 32; ++i) x[i] = seen ? __uint_as_float(v[i]) * inv : 0.0f;
                        if (real) {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                reinterpret_cast<uint4 *>(o)[4 * c + i] =
                                    make_uint4(ph_bits(__floats2half2_rn(x[8 * i], x[8 * i + 2])),
                                               ph_bits(__floats2half2_rn(x[8 * i + 1], x[8 * i + 3])),
                                               ph_bits(__floats2half2_rn(x[8 * i + 4], x[8 * i + 6])),
                                               ph_bits(__floats2half2_rn(x[8 * i + 5], x[8 * i + 7])));
                        }
                    }
                    if (real && a.lse)
                        a.lse[(static_cast<int64_t>(b) * a.NH + h) * a.T + t] =
                            seen ? (m + log2f(l)) * 0.6931471805599453f : -INFINITY;
                }
            }
        } else if (warp < 16) {
            // ================================================== expansion: a warp 16 keys, so one page and one scale
            fewer_registers<72>();
            constexpr int kPerRow = D / 16, kRows = 32 / kPerRow, kPasses = 16 / kRows;
            const int slice = warp - 8;
            // Eight lanes write a unit of two rows' quarters: every bank once per store instruction
            const int c = D == 128 ? (lane & 3) + 4 * ((lane >> 3) & 1) : lane & 3;
            const int r0 = D == 128 ? ((lane >> 2) & 1) + 2 * (lane >> 4) : lane >> 2;
            const int32_t *bt = a.table + b * a.t_stride;
            const int64_t lane_off = head * a.pg.head_stride + r0 * a.pg.row_stride + 16 * c;
            const int page_mask = (1 << a.pg.page_log2) - 1;
            int64_t key = static_cast<int64_t>(tile0) * kPKeys + 16 * slice;  // the slice's first key
            const auto look = [&](int64_t k) { return k < n ? max(kv8_page(a.pg, bt, k), 0) : 0; };
            const auto fetch = [&](const int8_t *codes, int64_t k, int page, uint4 *x) {
                const int8_t *at = codes + page * a.pg.page_stride + (static_cast<int>(k) & page_mask) * a.pg.row_stride + lane_off;
                const int64_t left = n - k - r0;  // keys past the end: value 0, and hidden
#pragma unroll
                for (int i = 0; i < kPasses; ++i) {
                    x[i] = make_uint4(0, 0, 0, 0);
                    if (i * kRows < left) x[i] = ldg_nc_v4(at);
                    at += kRows * a.pg.row_stride;
                }
            };
            const uint32_t at0 = unit_at(16 * slice + r0, 2 * c), at1 = unit_at(16 * slice + r0, 2 * c + 1);
            const auto expand = [&](uint32_t tile, const uint4 *x) {
#pragma unroll
                for (int i = 0; i < kPasses; ++i) {
                    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
                    uint32_t v[8];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        __half2 even, odd;
                        kv8_unpack(w[e], even, odd);
                        v[2 * e] = ph_bits(even);
                        v[2 * e + 1] = ph_bits(odd);
                    }
                    // kRows rows on: for D = 128 the swizzle's row bits change with every second pass
                    const uint32_t flip = D == 128 ? static_cast<uint32_t>((4 * i) & 4) << 4 : 0u;
                    sts128(tile + (at0 ^ flip) + i * kRows * 128, v[0], v[1], v[2], v[3]);
                    sts128(tile + (at1 ^ flip) + i * kRows * 128, v[4], v[5], v[6], v[7]);
                }
            };
            uint4 kx[kPasses], vx[kPasses];
            // pages are looked up two tiles ahead, scales and codes one
            int page = look(key), ahead = look(key + kPKeys);
            fetch(a.pg.k, key, page, kx);
            fetch(a.pg.v, key, page, vx);
            __half ks, vs;
            const auto scales = [&](int64_t k, int pg) {
                const int64_t so = k < n ? kv8_scale_offset(a.pg, pg, head, k) : 0;
                ks = a.pg.ks[so];
                vs = a.pg.vs[so];
            };
            scales(key, page);
            for (int j = 0; j < tiles; ++j) {
                const int st = j & 1;
                if (lane == 0) {  // the factors of these 16 keys (the ring of 4 outlives their readers)
                    // a block of scale 0 has values 0: the least scale's exponent moves no reference.  One of NaN is taken
                    // alike, so that the softmax's statistics, which are the scores' alone, stay theirs; rows that see it
                    // get NaN at the end.
                    const bool some = key < n;
                    float v = some ? __half2float(vs) : 0.0f;
                    const float kf = some ? __half2float(ks) * a.scale_log2 : 0.0f;
                    if (v != v) {
                        atomicMin(nan_from, static_cast<int>(key));
                        v = 0.0f;
                    }
                    const float lv = v == 0.0f ? -24.0f : log2f(v);
                    meta[(j & 3) * 8 + slice] = make_ulonglong2(f32x2(kf, kf), f32x2(lv, lv));
                    inv_vs[(j & 3) * 8 + slice] = v == 0.0f ? 16777216.0f : 1.0f / v;
                    mbar_arrive(&meta_full[j & 3]);
                }
                key += kPKeys;
                page = ahead;
                if (j + 1 < tiles) {
                    scales(key, page);
                    ahead = look(key + kPKeys);
                }
                if (j >= 2) mbar_wait_or(&k_free[st], ((j >> 1) - 1) & 1, stop);
                expand(base + S::kK + st * S::kTile, kx);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&k_full[st]);
                if (j + 1 < tiles) fetch(a.pg.k, key, page, kx);
                if (j >= 2) mbar_wait_or(&v_free[st], ((j >> 1) - 1) & 1, stop);
                expand(base + S::kV + st * S::kTile, vx);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&v_full[st]);
                if (j + 1 < tiles) fetch(a.pg.v, key, page, vx);
            }
        } else {
            fewer_registers<64>();
            if (warp == 16) {
                // ============================================== MMA: the warp waits together, one lane issues.  What the
                // instructions take is made warp-uniform by reductions, so that it lives in uniform registers.
                const uint32_t tm = __reduce_max_sync(0xffffffffu, tmem);
                const int nt = __reduce_max_sync(0xffffffffu, tiles);
                const uint32_t idesc_s = umma_idesc(128, 128, false), idesc_o = umma_idesc(128, D, true);
                const auto scores = [&](int buf, int qi, int st) {
                    const uint32_t q = umma_desc_lo(base + S::kQ + qi * S::kTile);
                    const uint32_t k = umma_desc_lo(base + S::kK + st * S::kTile);
#pragma unroll
                    for (int s = 0; s < D / 16; ++s) {
                        const uint32_t off = static_cast<uint32_t>((s >> 2) * 1024 + 2 * (s & 3));  // 16-byte units
                        umma_ss(tm + 128 * buf, q + off, k + off, idesc_s, s > 0);
                    }
                    umma_commit(&s_ready[buf]);
                    if (qi == 1) umma_commit(&k_free[st]);
                };
                const auto values = [&](int buf, int qi, int st, bool acc) {
                    const uint32_t v = umma_desc_lo(base + S::kV + st * S::kTile, 16384);
#pragma unroll
                    for (int s = 0; s < 8; ++s)
                        umma_ts(tm + S::kO + D * qi, tm + 128 * buf + 8 * s, v + 128 * s, idesc_o, acc || s > 0);
                };
                mbar_wait_or(q_full, 0, stop);
#pragma unroll
                for (int i = 0; i < S::kS; ++i) {  // the first S of every buffer
                    if (i >> 1 >= nt) break;
                    if ((i & 1) == 0) mbar_wait_or(&k_full[i >> 1], 0, stop);
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if (elect_one()) scores(i, i & 1, i >> 1);
                    __syncwarp();
                }
                // P V of number 2 j + qi, then the S that is kS numbers on over it
                int buf = 0, turn = 0;
                for (int j = 0; j < nt; ++j) {
                    const int st = j & 1;
                    mbar_wait_or(&v_full[st], (j >> 1) & 1, stop);
                    if (S::kS == 2 && j + 1 < nt) mbar_wait_or(&k_full[st ^ 1], ((j + 1) >> 1) & 1, stop);
#pragma unroll
                    for (int qi = 0; qi < 2; ++qi) {
                        const int at = S::kS == 2 ? qi : buf, on = S::kS == 2 ? qi : qi ^ 1, ahead = j + (qi + S::kS) / 2;
                        mbar_wait_or(&p_ready[at], S::kS == 2 ? j & 1 : turn, stop);
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        if (elect_one()) {
                            values(at, qi, st, j > 0);
                            if (qi == 1) umma_commit(&v_free[st]);
                            if (S::kS > 2) umma_commit(&o_added[qi]);
                            if (S::kS == 2 && ahead < nt) scores(at, on, ahead & 1);
                        }
                        __syncwarp();
                        if (S::kS > 2 && ahead < nt) {
                            if (on == 0) mbar_wait_or(&k_full[ahead & 1], (ahead >> 1) & 1, stop);
                            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                            if (elect_one()) scores(at, on, ahead & 1);
                            __syncwarp();
                        }
                        if (++buf == S::kS) buf = 0, turn ^= 1;
                    }
                }
                if (elect_one()) umma_commit(o_done);
                __syncwarp();
                *stop_last = 0;
                mbar_wait_or(o_done, 0, stop_last);  // nothing of this CTA is in flight when it frees its TMEM
            }
        }
    } else if (warp < 8 && a.splits == 1) {
        // no query of the pair sees a key: zeros
        const int qi = warp >> 2, row = tid & 127;
        const int t = t_first + qi * TT + row / group, h = head * group + row % group;
        if (row < TT * group && t < a.T) {
            uint4 *o = reinterpret_cast<uint4 *>(a.out + b * a.o_sb + static_cast<int64_t>(t) * a.o_st + h * a.o_sh);
            for (int i = 0; i < D / 8; ++i) o[i] = make_uint4(0, 0, 0, 0);
            if (a.lse) a.lse[(static_cast<int64_t>(b) * a.NH + h) * a.T + t] = -INFINITY;
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (tid == 0 && *stop) report_device_error(T2C_ETIMEOUT);
    if (warp == 16) {
        __syncwarp();
        tmem_free(tmem, 512);
    }
}

// Joins the splits, a warp per query row: 7 us for 45 queries of 32 heads in 18 splits, 13 MB.
template <int D>
__global__ void __launch_bounds__(256) attn8_prefill_join_kernel(const __grid_constant__ PrefillArgs a) {
    const int lane = threadIdx.x & 31;
    const unsigned w = blockIdx.x * 8u + (threadIdx.x >> 5), tokens = w / static_cast<unsigned>(a.NH);
    if (tokens >= static_cast<unsigned>(a.B) * a.T) return;
    const int h = static_cast<int>(w % a.NH), t = static_cast<int>(tokens % a.T), b = static_cast<int>(tokens / a.T);
    const int group = a.NH / a.pg.n_kv, TT = kPRows / group, head = h / group;
    const int pair = t / (2 * TT), in_pair = t % (2 * TT);
    const int row = in_pair / TT * 128 + in_pair % TT * group + h % group;
    const int64_t p0 = a.positions[b];
    const int64_t n = min(p0 + min(pair * 2 * TT + 2 * TT, a.T), a.max_len);  // as the CTA had it
    const int tiles = n > 0 ? static_cast<int>((n + kPKeys - 1) / kPKeys) : 0;
    const int per = (tiles + a.splits - 1) / a.splits, used = per > 0 ? (tiles + per - 1) / per : 0;
    const float *base = a.parts + ((static_cast<int64_t>(b) * a.pg.n_kv + head) * a.pairs + pair) * a.splits * (256 * (D + 2));
    const bool seen = p0 + t >= 0;
    // positions were there before the kernel whose parts are joined: all of the above runs under that one's end
    pdl_wait();
    pdl_trigger();
    constexpr int kPer = D / 32, kAhead = 8;
    constexpr int64_t kPart = 256 * (D + 2);
    // lane s (and s + 32): the statistics of split s; the first rows of O come beside them
    using Vec = typename std::conditional<kPer == 4, float4, float2>::type;
    const float *rows = base + row * D + kPer * lane;
    Vec v[kAhead];
#pragma unroll
    for (int s = 0; s < kAhead; ++s)
        if (s < used) v[s] = *reinterpret_cast<const Vec *>(rows + s * kPart);
    float m[2], l[2], top = kPRefStart;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int s = lane + 32 * k;
        m[k] = s < used ? base[s * kPart + 256 * D + row] : kPRefStart;
        l[k] = s < used ? base[s * kPart + 256 * (D + 1) + row] : 0.0f;
        top = fmaxf(top, m[k]);
    }
    top = warp_max(top);
    float f[2] = {ex2(m[0] - top), ex2(m[1] - top)};
    const float sum = warp_sum(fmaf(l[0], f[0], l[1] * f[1]));
    float acc[kPer] = {};
    for (int s0 = 0; s0 < used; s0 += kAhead) {
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int s = s0 + k;
            const float w = __shfl_sync(0xffffffffu, s < 32 ? f[0] : f[1], s & 31);
            const float *o = reinterpret_cast<const float *>(&v[k]);
#pragma unroll
            for (int i = 0; i < kPer; ++i)
                if (s < used) acc[i] = fmaf(o[i], w, acc[i]);
            if (s + kAhead < used) v[k] = *reinterpret_cast<const Vec *>(rows + (s + kAhead) * kPart);
        }
    }
    const float inv = seen ? 1.0f / sum : 0.0f;
    __half2 *out = reinterpret_cast<__half2 *>(a.out + b * a.o_sb + static_cast<int64_t>(t) * a.o_st + h * a.o_sh) + kPer / 2 * lane;
#pragma unroll
    for (int i = 0; i < kPer / 2; ++i)
        out[i] = seen ? __floats2half2_rn(acc[2 * i] * inv, acc[2 * i + 1] * inv) : __float2half2_rn(0.0f);
    if (a.lse && lane == 0)
        a.lse[(static_cast<int64_t>(b) * a.NH + h) * a.T + t] = seen ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
}

}  // namespace

cudaError_t status_attn8_tc(unsigned int *bits, int clear, cudaStream_t s) { return read_tu_status(bits, clear, s); }

}  // namespace t2c

using namespace t2c;

namespace {

struct PrefillPlan {
    int pairs, splits;
    int64_t floats;
};

// One CTA per SM: the keys of a pair of query tiles are split while CTAs would be missing, at least two tiles each.
// (45 queries on 9111 keys, 32 heads on 8: 18 splits 27 us; one 170, 9 35, 36 40.  512 on 8192: two splits 104 us, one
// 160, four 116.  4 x 512 on up to 3500, 16 heads of 64 on 16: one split 65, two 91.)
PrefillPlan prefill_plan(int64_t B, int64_t T, int64_t NH, int64_t NK, int64_t D, int64_t max_len, int64_t splits) {
    PrefillPlan r = {};
    const int64_t tokens = 2 * (kPRows / (NH / NK));
    r.pairs = static_cast<int>((T + tokens - 1) / tokens);
    const int64_t items = B * NK * r.pairs, tiles = (max_len + kPKeys - 1) / kPKeys;
    int64_t s = splits;
    if (s == 0) {
        s = sm_count() / items;
        s = s > tiles / 2 ? tiles / 2 : s;
    }
    s = s > 64 ? 64 : s;
    r.splits = static_cast<int>(s < 1 ? 1 : s);
    r.floats = r.splits > 1 ? items * r.splits * 256 * (D + 2) : 0;
    return r;
}

}  // namespace

extern "C" int64_t t2c_attn_prefill_q8_workspace(const t2c_q8_pages *pages, int64_t bt_width, int64_t B, int64_t T,
                                                 int64_t NH, int64_t max_len, int64_t splits) {
    if (!pages || pages->n_kv <= 0 || NH <= 0 || NH % pages->n_kv || NH / pages->n_kv > kPRows || B <= 0 || T <= 0 ||
        splits < 0 || bt_width <= 0)
        return -1;
    const int64_t capacity = bt_width * pages->page_size;
    if (max_len <= 0 || max_len > capacity) max_len = capacity;
    return prefill_plan(B, T, NH, pages->n_kv, pages->head_dim, max_len, splits).floats;
}

extern "C" int t2c_attn_prefill_q8(const t2c_q8_pages *pages, const void *q, int64_t q_sb, int64_t q_st, int64_t q_sh,
                                   void *out, int64_t o_sb, int64_t o_st, int64_t o_sh, float *lse,
                                   const int32_t *positions, const int32_t *block_table, int64_t bt_stride,
                                   int64_t bt_width, int64_t B, int64_t T, int64_t NH, float scale, int64_t max_len,
                                   int64_t splits, float *workspace, int64_t workspace_floats, void *stream) {
    PrefillArgs a = {};
    int rc = kv8_attn_check(pages, "attn_prefill_q8", a.pg, block_table, bt_stride, bt_width, positions, B, T, NH, max_len);
    if (rc != T2C_OK) return rc;
    if (!kv8_strides(q, B, q_sb, T, q_st, NH, q_sh) || !kv8_strides(out, B, o_sb, T, o_st, NH, o_sh))
        return set_error(T2C_EINVAL, "attn_prefill_q8: q and out rows must be 16-byte aligned");
    if (splits < 0) return set_error(T2C_EINVAL, "attn_prefill_q8: splits %lld", (long long)splits);
    const int64_t D = pages->head_dim;
    if (NH / a.pg.n_kv > kPRows) return set_error(T2C_EUNSUPPORTED, "attn_prefill_q8: group %lld", (long long)(NH / a.pg.n_kv));
    const PrefillPlan plan = prefill_plan(B, T, NH, a.pg.n_kv, D, max_len, splits);
    if (plan.floats > 0 && (!workspace || workspace_floats < plan.floats))
        return set_error(T2C_ESCRATCH, "attn_prefill_q8: workspace needs %lld floats", (long long)plan.floats);
    if (!kv8_aligned(workspace, 16)) return set_error(T2C_EINVAL, "attn_prefill_q8: workspace must be 16-byte aligned");
    a.q = static_cast<const __half *>(q), a.q_sb = q_sb, a.q_st = q_st, a.q_sh = q_sh;
    a.out = static_cast<__half *>(out), a.o_sb = o_sb, a.o_st = o_st, a.o_sh = o_sh;
    a.lse = lse;
    a.positions = positions, a.table = block_table, a.t_stride = bt_stride, a.max_len = max_len;
    a.B = static_cast<int>(B), a.T = static_cast<int>(T), a.NH = static_cast<int>(NH);
    a.pairs = plan.pairs, a.splits = plan.splits;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.parts = workspace;
    const int64_t ctas = B * a.pg.n_kv * plan.pairs * plan.splits, rows = B * T * NH;
    if (ctas > INT32_MAX || rows > UINT32_MAX - 8) return set_error(T2C_EINVAL, "attn_prefill_q8: bad shape");
    const cudaStream_t s = as_stream(stream);
    const auto kern = D == 128 ? attn8_prefill_kernel<128> : attn8_prefill_kernel<64>;
    const int smem = D == 128 ? PrefillShape<128>::kSmem : PrefillShape<64>::kSmem;
    rc = kv8_configure(kern, smem, D == 128 ? 2 : 3, "attn_prefill_q8");
    if (rc == T2C_OK) rc = kv8_launch("attn_prefill_q8", kern, dim3(static_cast<unsigned>(ctas)), dim3(kPThreads), smem, 1, s, a);
    if (rc != T2C_OK || plan.splits == 1) return rc;
    return kv8_launch("attn_prefill_q8 join", D == 128 ? attn8_prefill_join_kernel<128> : attn8_prefill_join_kernel<64>,
                      dim3(static_cast<unsigned>((rows + 7) / 8)), dim3(256), 0, 1, s, a);
}
