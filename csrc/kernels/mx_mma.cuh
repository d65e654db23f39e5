// Block-scaled tcgen05.mma and what feeds it, shared by the microscaled products: operand kinds, descriptors, scale
// copies, predicated asynchronous instructions, tensor maps of codes and scales.
#pragma once

#include <cudaTypedefs.h>

#include "microscale.cuh"
#include "tcgen05.cuh"

namespace mmltk {
namespace mx {

using namespace tc;

constexpr int kRowBytes = 128;                     // bytes of codes per row and stage

template <MxFormat F>
struct Kind;
template <>
struct Kind<MxFormat::kMxFp4> {
    static constexpr int kAtoms = 2, kElems = 256;     // scale tiles and elements of a stage
    static constexpr uint32_t kDesc = (1u << 7) | (1u << 10) | (1u << 23);   // e2m1 x e2m1, e8m0 scales
};
template <>
struct Kind<MxFormat::kNvFp4> {
    static constexpr int kAtoms = 4, kElems = 256;
    static constexpr uint32_t kDesc = (1u << 7) | (1u << 10);                // e2m1 x e2m1, e4m3 scales
};
template <>
struct Kind<MxFormat::kMxFp8> {
    static constexpr int kAtoms = 1, kElems = 128;
    static constexpr uint32_t kDesc = 1u << 23;                              // e4m3 x e4m3, e8m0 scales
};

// The loading and the issuing warp run their loops with all lanes and predicate the asynchronous instructions on
// one elected lane: operands then live in uniform registers.  (In a one-lane branch every operand is
// moved there first, and the ~16 instructions of a stage took the issuing thread about 900 cycles.)
__device__ __forceinline__ uint32_t elect_lane() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p;
}

__device__ __forceinline__ uint32_t mbar_test(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return ok;
}

// Upper halves of the shared-memory descriptors: 128-byte swizzled K-major operand (8-row groups 1024 bytes
// apart), and unswizzled 32 x 16 byte scale tile (8-row groups 128 bytes apart).
constexpr uint32_t kOperandHi = (1024u >> 4) | (1u << 14) | (2u << 29);
constexpr uint32_t kScaleHi = (128u >> 4) | (1u << 14);
// lower halves
__device__ __forceinline__ uint32_t operand_lo(uint32_t addr) { return (addr >> 4) | (1u << 16); }

#define MMLTK_MX_MMA(group, kind)                                                                                   \
    asm volatile("{\n\t.reg .pred p, e;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 e, %0, 0;\n\tsetp.ne.b32 p, %7, 0;\n\t"    \
                 "mov.b64 da, {%2, %8};\n\tmov.b64 db, {%3, %8};\n\t"                                                \
                 "@e tcgen05.mma.cta_group::" group ".kind::" kind " [%1], da, db, %4, [%5], [%6], p;\n\t}" ::"r"(elected), \
                 "r"(d), "r"(a), "r"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "n"(kOperandHi)           \
                 : "memory")
template <MxFormat F, bool kPair>
__device__ __forceinline__ void mma_block(uint32_t elected, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                          uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
    if constexpr (F == MxFormat::kNvFp4) {
        if constexpr (kPair) MMLTK_MX_MMA("2", "mxf4nvf4.block_scale.scale_vec::4X");
        else MMLTK_MX_MMA("1", "mxf4nvf4.block_scale.scale_vec::4X");
    } else if constexpr (F == MxFormat::kMxFp4) {
        if constexpr (kPair) MMLTK_MX_MMA("2", "mxf4.block_scale.scale_vec::2X");
        else MMLTK_MX_MMA("1", "mxf4.block_scale.scale_vec::2X");
    } else {
        if constexpr (kPair) MMLTK_MX_MMA("2", "mxf8f6f4.block_scale.scale_vec::1X");
        else MMLTK_MX_MMA("1", "mxf8f6f4.block_scale.scale_vec::1X");
    }
}
#undef MMLTK_MX_MMA

// One 32 x 16 byte scale tile (lo = address / 16) from shared memory to 4 columns of tensor memory, in all four lane
// quarters (of each CTA of a pair, from its own shared memory).
template <bool kPair>
__device__ __forceinline__ void copy_scales(uint32_t elected, uint32_t taddr, uint32_t lo) {
    if constexpr (kPair)
        asm volatile(
            "{\n\t.reg .pred e;\n\t.reg .b64 d;\n\tsetp.ne.b32 e, %0, 0;\n\tmov.b64 d, {%2, %3};\n\t"
            "@e tcgen05.cp.cta_group::2.32x128b.warpx4 [%1], d;\n\t}" ::"r"(elected), "r"(taddr), "r"(lo), "n"(kScaleHi)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred e;\n\t.reg .b64 d;\n\tsetp.ne.b32 e, %0, 0;\n\tmov.b64 d, {%2, %3};\n\t"
            "@e tcgen05.cp.cta_group::1.32x128b.warpx4 [%1], d;\n\t}" ::"r"(elected), "r"(taddr), "r"(lo), "n"(kScaleHi)
            : "memory");
}
template <bool kPair>
__device__ __forceinline__ void commit(uint32_t elected, uint32_t bar) {
    if constexpr (kPair)
        asm volatile(
            "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %0, 0;\n\t"
            "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%1];\n\t}" ::"r"(elected), "r"(bar)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %0, 0;\n\t"
            "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n\t}" ::"r"(elected), "r"(bar)
            : "memory");
}

// Tensor loads whose completion counts on the barrier `bar` (shared::cluster address; a pair's is the even CTA's).
#define MMLTK_MX_LOAD(form, coords, ...)                                                                           \
    asm volatile("{\n\t.reg .pred e;\n\tsetp.ne.b32 e, %0, 0;\n\t"                                                  \
                 "@e cp.async.bulk.tensor." form ".shared::cluster.global.mbarrier::complete_tx::bytes [%1], [%2, " coords \
                 "], [%3];\n\t}" ::"r"(elected),                                                                   \
                 "r"(dst), "l"(map), "r"(bar), __VA_ARGS__                                                         \
                 : "memory")
template <bool kPair>
__device__ __forceinline__ void load_2d(uint32_t elected, const CUtensorMap* map, uint32_t bar, uint32_t dst, int c0,
                                        int c1) {
    if constexpr (kPair) MMLTK_MX_LOAD("2d.cta_group::2", "{%4, %5}", "r"(c0), "r"(c1));
    else MMLTK_MX_LOAD("2d", "{%4, %5}", "r"(c0), "r"(c1));
}
template <bool kPair>
__device__ __forceinline__ void load_3d(uint32_t elected, const CUtensorMap* map, uint32_t bar, uint32_t dst, int c0,
                                        int c1, int c2) {
    if constexpr (kPair) MMLTK_MX_LOAD("3d.cta_group::2", "{%4, %5, %6}", "r"(c0), "r"(c1), "r"(c2));
    else MMLTK_MX_LOAD("3d", "{%4, %5, %6}", "r"(c0), "r"(c1), "r"(c2));
}
#undef MMLTK_MX_LOAD

// The factor g_x g_w of a sum.  Where the product of the two tensor scales is no normal number although a sum times both
// may be one (inputs of 1e-18 on either side; a sum of zeros between large ones), a power of two goes to the sum
// first, which is exact.  Scales found from data are 2^-100 to 2^117.
struct Alpha {
    float pre, rest;
};
__device__ __forceinline__ Alpha product_scale(const float* x_g, const float* w_g) {
    const float x = x_g ? *x_g : 1.f, w = w_g ? *w_g : 1.f, a = x * w;
    if (fabsf(a) >= 1.17549435e-38f && fabsf(a) <= 3.402823466e38f) return {1.f, a};
    const float lo = fabsf(x) < fabsf(w) ? x : w, hi = fabsf(x) < fabsf(w) ? w : x;
    if (fabsf(a) < 1.f) return {1.2621774483536189e-29f, lo * 7.9228162514264338e28f * hi};      // 2^-96
    return {5.1922968585348276e33f, hi * 1.9259299443872359e-34f * lo};                          // 2^112
}

inline PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    }();
    return fn;
}

// Codes: bytes [rows, row_bytes] (pitch), boxes of 128 bytes x box_rows, 128-byte swizzle, zero fill.
inline bool codes_map(CUtensorMap* map, const void* p, int64_t row_bytes, int64_t rows, int64_t pitch, int box_rows) {
    auto fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(row_bytes), static_cast<cuuint64_t>(rows)};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch)};
    cuuint32_t box[2] = {kRowBytes, static_cast<cuuint32_t>(box_rows)}, es[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), dims, strides, box, es,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Scales: [row tiles, tiles along k, 512 bytes], boxes of `atoms` tiles x `row_tiles`.
inline bool scales_map(CUtensorMap* map, const void* p, int64_t rows, int kt, int atoms, int row_tiles) {
    auto fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[3] = {256, static_cast<cuuint64_t>(kt), static_cast<cuuint64_t>((rows + 127) / 128)};
    cuuint64_t strides[2] = {512, static_cast<cuuint64_t>(kt) * 512};
    cuuint32_t box[3] = {256, static_cast<cuuint32_t>(atoms), static_cast<cuuint32_t>(row_tiles)}, es[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(p), dims, strides, box, es,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace mx
}  // namespace mmltk
