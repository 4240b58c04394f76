// Paged KV cache in 8 bits: the device view of the pool and the code <-> value
// helpers that the write, read, eviction and attention kernels share.
//
// A code c (int8, -127..127) of a block of `block` consecutive tokens of one
// KV head stands for c * s, s the block's fp16 scale.  c * s has at most
// 7 + 11 significant bits, so fp32 holds it exactly.  A NaN scale marks a block
// that was given a non-finite value: all of it reads as NaN.
#pragma once

#include <cudaTypedefs.h>
#include <math.h>

#include "common.cuh"
#include "umma.cuh"

namespace t2c {

struct KvPages {
    int8_t *k, *v;
    __half *ks, *vs;
    int64_t page_stride, head_stride, row_stride;  // codes, in elements (= bytes)
    int64_t s_page_stride, s_head_stride;          // scales, in elements
    int num_pages, n_kv, page_log2, block_log2;
};

// Checks the pool's description; fills `out`.  `what` names the entry point in messages.
int kv8_view(const t2c_q8_pages *pages, const char *what, KvPages &out);
// Checks a block table against the pool: returns T2C_OK and the capacity in positions.
int kv8_table(const t2c_q8_pages *pages, const int32_t *table, int64_t B, int64_t stride, int64_t width, const char *what,
              int64_t &capacity);

// What the attention entry points check alike; max_len becomes the bound in positions.
int kv8_attn_check(const t2c_q8_pages *pages, const char *what, KvPages &pg, const int32_t *table, int64_t bt_stride,
                   int64_t bt_width, const int32_t *positions, int64_t B, int64_t T, int64_t NH, int64_t &max_len);

// cuTensorMapEncodeTiled, or null.
PFN_cuTensorMapEncodeTiled kv8_encoder();

// Tensor maps of the codes as (dim, row of page, KV head, page), boxes of `rows` rows of one head in the swizzle that
// is as wide as a row (128 or 64 bytes).  False when the driver refuses.
bool kv8_maps(const t2c_q8_pages *pages, int rows, CUtensorMap &k_map, CUtensorMap &v_map);

// A box of the codes at (row, head, page) into shared memory (no multicast).
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int w, uint64_t *bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::
            "r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
        : "memory");
}

// Physical page of a position; an entry outside the pool is reported and becomes -1.
__device__ __forceinline__ int kv8_page(const KvPages &pg, const int32_t *__restrict__ table, int64_t pos) {
    const int page = table[pos >> pg.page_log2];
    if (static_cast<unsigned>(page) < static_cast<unsigned>(pg.num_pages)) return page;
    report_device_error(T2C_EINVAL);
    return -1;
}

__device__ __forceinline__ int64_t kv8_row_offset(const KvPages &pg, int page, int head, int64_t pos) {
    return page * pg.page_stride + head * pg.head_stride + (pos & ((1 << pg.page_log2) - 1)) * pg.row_stride;
}

__device__ __forceinline__ int64_t kv8_scale_offset(const KvPages &pg, int page, int head, int64_t pos) {
    return page * pg.s_page_stride + head * pg.s_head_stride + ((pos & ((1 << pg.page_log2) - 1)) >> pg.block_log2);
}

// Four codes (one 32-bit word) as two half2, exactly: the biased byte c + 128 placed in the low mantissa
// bits of 1024 gives 1152 + c, and the subtraction is exact.  even = codes 0 and 2, odd = codes 1 and 3.
__device__ __forceinline__ void kv8_unpack(uint32_t w, __half2 &even, __half2 &odd) {
    uint32_t lo, hi;
    asm("{\n .reg .b32 m, x;\n mov.b32 m, 0x00ff00ff;\n mov.b32 x, 0x64806480;\n lop3.b32 %0, %1, m, x, 0x6a;\n}\n" : "=r"(lo) : "r"(w));
    asm("{\n .reg .b32 m, x;\n mov.b32 m, 0x00ff00ff;\n mov.b32 x, 0x64806480;\n lop3.b32 %0, %1, m, x, 0x6a;\n}\n" : "=r"(hi) : "r"(w >> 8));
    const __half2 bias = __half2half2(__ushort_as_half(0x6480));  // 1152
    even = __hsub2(*reinterpret_cast<const __half2 *>(&lo), bias);
    odd = __hsub2(*reinterpret_cast<const __half2 *>(&hi), bias);
}

// Least fp16 scale with 127 * s >= top, at most 515.5 (127 * 515.5 is the largest such product that fp16
// holds; the fp16 values above it still get code 127).  top / 127 in fp32 picks the right fp16 neighbour: the
// quotient of an at most 18-bit number by 127 is either an fp16 number or differs from one by more than 2^-20
// of itself.  top = +inf (a non-finite value was seen) gives NaN.
__device__ __forceinline__ __half kv8_scale_for(float top) {
    if (!(top < INFINITY)) return __ushort_as_half(0x7fff);
    return __float2half_ru(fminf(__fdiv_rn(top, 127.0f), 515.5f));
}

__device__ __forceinline__ uint32_t kv8_pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// Largest and least code of a word's four, folded into running s16x2 extremes.
__device__ __forceinline__ void kv8_extremes(uint32_t w, uint32_t &most, uint32_t &least) {
    uint32_t even, odd;  // bytes 0, 2 and 1, 3, sign-extended
    asm("prmt.b32 %0, %1, 0, 0xa280;" : "=r"(even) : "r"(w));
    asm("prmt.b32 %0, %1, 0, 0xb391;" : "=r"(odd) : "r"(w));
    most = __vimax3_s16x2(even, odd, most);
    least = __vimin3_s16x2(even, odd, least);
}

__device__ __forceinline__ int kv8_largest(uint32_t most, uint32_t least) {
    const auto half = [](uint32_t v, int h) { return static_cast<int>(static_cast<int16_t>(v >> (16 * h))); };
    return max(max(half(most, 0), half(most, 1)), -min(half(least, 0), half(least, 1)));
}

// x / s in two floats, high + low to 2^-46 of it (inv = 1 / s).
__device__ __forceinline__ float2 kv8_ratio(float x, float s, float inv) {
    const float high = __fdiv_rn(x, s);
    return make_float2(high, fmaf(-high, s, x) * inv);
}

// rint of two values times a ratio, |result| <= 127, as the low bytes of two words.  With a code of 7 bits and ratios of two
// scales of 11, or a value of 11 bits and one over a scale, this is the correctly rounded quotient: the small product first,
// what is rounded is within 2^-23 of the quotient, whose distance from a tie is zero or at least 2^-19 of it, and it is the
// quotient itself where that is a tie.  1.5 * 2^23 then leaves the integer in the low mantissa bits.
__device__ __forceinline__ uint64_t kv8_codes(uint64_t x, float2 ratio) {
    const uint64_t y = f32x2_fma(x, f32x2(ratio.x, ratio.x), f32x2_mul(x, f32x2(ratio.y, ratio.y)));
    return f32x2_add(y, f32x2(12582912.0f, 12582912.0f));
}

__device__ __forceinline__ uint32_t kv8_pack(uint64_t a, uint64_t b) {
    const float2 x = f32x2_parts(a), y = f32x2_parts(b);
    return kv8_pack4(__float_as_uint(x.x), __float_as_uint(x.y), __float_as_uint(y.x), __float_as_uint(y.y));
}

// A word's four codes at another scale.  (Code + 128 in the mantissa of 2^23 becomes a float without a conversion
// instruction, two values an instruction from there on.  With conversions, and product, quotient and its correction for each
// code, the move of 4 x 4096 rows of 8 heads ran 17 M instructions instead of 13 M, in place 55 us instead of 49.)
__device__ __forceinline__ uint32_t kv8_recode(uint32_t w, float2 ratio) {
    const uint32_t u = w ^ 0x80808080u;
    const uint64_t bias = f32x2(-8388736.0f, -8388736.0f);
    uint64_t c[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        c[i] = kv8_codes(f32x2_add(f32x2(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 + 2 * i)),
                                         __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441 + 2 * i))), bias), ratio);
    return kv8_pack(c[0], c[1]);
}

// overlap: the kernel may be resident before the one ahead of it in the stream has ended (it waits in pdl_wait).
template <typename Kernel, typename... Args>
int kv8_launch_as(bool overlap, const char *what, Kernel kernel, dim3 grid, dim3 block, size_t smem, unsigned cluster,
                  cudaStream_t stream, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = overlap ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, args...);
    if (err != cudaSuccess) return set_error(T2C_ECUDA, "%s launch: %s", what, cudaGetErrorString(err));
    return T2C_OK;
}

template <typename Kernel, typename... Args>
int kv8_launch(const char *what, Kernel kernel, dim3 grid, dim3 block, size_t smem, unsigned cluster, cudaStream_t stream,
               Args... args) {
    return kv8_launch_as(true, what, kernel, grid, block, smem, cluster, stream, args...);
}

// Raises a kernel's shared-memory limit once per device; `slot` numbers the kernel.
template <typename Kernel>
int kv8_configure(Kernel kern, int smem, int slot, const char *what) {
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

inline bool kv8_aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// An fp16 tensor whose rows are 16-byte aligned: (entries, stride) of its dimensions but the last.  One entry has no stride.
inline bool kv8_strides(const void *p, int64_t na, int64_t a, int64_t nb, int64_t b, int64_t nc, int64_t c) {
    const auto fits = [](int64_t n, int64_t stride) { return n == 1 || stride % 8 == 0; };
    return p && kv8_aligned(p, 16) && fits(na, a) && fits(nb, b) && fits(nc, c);
}

}  // namespace t2c
