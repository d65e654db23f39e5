// Microscaled number formats: a block of consecutive elements of a row shares one scale byte.
//
//   mxfp4  e2m1 elements (largest 6), 32 per scale, scale = a power of two (e8m0)
//   nvfp4  e2m1 elements, 16 per scale, scale = e4m3, times one fp32 scale g of the whole tensor
//   mxfp8  e4m3 elements (largest 448), 32 per scale, scale = a power of two (e8m0)
//
// Codes: 4-bit elements two to a byte, the even element in the low half; rows padded to 16 bytes.
// Scales: tiles of 128 rows x 4 blocks (512 bytes), byte [r / 128][b / 4][r % 32][(r / 32) % 4][b % 4]
// for row r, block b, so that one tile is the 32 x 16 byte matrix that tcgen05.cp spreads over
// the 32 lanes of tensor memory; rows and blocks past the end are zero bytes.
#pragma once

#include <cuda_fp4.h>
#include <cuda_fp8.h>

#include <atomic>

#include "common.cuh"
#include "microscale.h"

namespace mmltk {
namespace mx {

template <MxFormat F>
struct Traits;
template <>
struct Traits<MxFormat::kMxFp4> {
    static constexpr int kBlock = 32, kBits = 4;
    static constexpr bool kPow2 = true;
};
template <>
struct Traits<MxFormat::kNvFp4> {
    static constexpr int kBlock = 16, kBits = 4;
    static constexpr bool kPow2 = false;
};
template <>
struct Traits<MxFormat::kMxFp8> {
    static constexpr int kBlock = 32, kBits = 8;
    static constexpr bool kPow2 = true;
};

// Offset of the scale byte of row r, block b in the tiled layout with kt = ceil(blocks / 4) tiles along a row.
__device__ __forceinline__ int64_t scale_offset(int64_t r, int b, int kt) {
    return ((r >> 7) * kt + (b >> 2)) * 512 + (r & 31) * 16 + ((r >> 5) & 3) * 4 + (b & 3);
}

struct BlockScale {
    uint32_t byte;   // the stored scale
    float inv;       // what x is multiplied with before it is rounded to an element
};

// Power-of-two scale: the smallest 2^p whose 2^p * (largest element) is not below amax, so no element
// saturates.  amax = 1.M * 2^(E - 127) against 1.5 * 2^2 (e2m1) or 1.75 * 2^8 (e4m3), on the bits;
// clamped at 2^-127.  A block with an infinity or NaN gets the NaN scale (0xff): its values read back NaN
// whatever their codes (zero for its finite elements and its padding; that of a NaN for the others).
template <int kBits>
__device__ __forceinline__ BlockScale pow2_scale(float amax) {
    const uint32_t u = __float_as_uint(amax);
    BlockScale s;
    if (u >= 0x7f800000u) {
        s.byte = 0xff;
        s.inv = 0.f;
        return s;
    }
    const int e = static_cast<int>(u >> 23), m = static_cast<int>(u & 0x7fffffu);
    const int p = kBits == 4 ? e - 2 + (m > 0x400000) : e - 8 + (m > 0x600000);
    s.byte = static_cast<uint32_t>(max(p, 0));
    s.inv = __uint_as_float((254u - s.byte) << 23);   // 2^-(byte - 127): byte <= 253, a normal number
    return s;
}

// e4m3 scale of amax / 6 on the tensor scale's grid; the elements are x times the rounded reciprocal
// 1 / (s g) (one division per block instead of one per element).  s = 0 (amax below 2^-10 * 6 g): all zero.
__device__ __forceinline__ BlockScale e4m3_scale(float amax, float g) {
    BlockScale s;
    if (__float_as_uint(amax) >= 0x7f800000u) {
        s.byte = 0x7f;
        s.inv = 0.f;
        return s;
    }
    const float t = fminf(amax / (6.0f * g), 448.0f);
    const __nv_fp8_storage_t q = __nv_cvt_float_to_fp8(t, __NV_SATFINITE, __NV_E4M3);
    s.byte = q;
    const float v = __half2float(__half(__nv_cvt_fp8_to_halfraw(q, __NV_E4M3)));
    s.inv = v > 0.f ? 1.0f / (v * g) : 0.f;
    return s;
}

template <MxFormat F>
__device__ __forceinline__ BlockScale block_scale(float amax, float g) {
    if constexpr (Traits<F>::kPow2) {
        return pow2_scale<Traits<F>::kBits>(amax);
    } else {
        return e4m3_scale(amax, g);
    }
}

// max that keeps a NaN (fmaxf drops it): on the bits of |x|, where NaN > infinity > every number
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ float max3_abs_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

__device__ __forceinline__ uint32_t cvt_e4m3x2(float lo, float hi) {
    return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t cvt_e2m1x2(float lo, float hi) {
    return __nv_cvt_float2_to_fp4x2(make_float2(lo, hi), __NV_E2M1, cudaRoundNearest);
}
// products of neighbours with one factor, two an instruction
__device__ __forceinline__ float2 scale2(const float* v, float inv) {
    float2 r;
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %4};\n\tmul.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(v[0]), "f"(v[1]), "f"(inv));
    return r;
}
__device__ __forceinline__ uint32_t cvt_e4m3x4(const float* v, float inv) {
    const float2 a = scale2(v, inv), b = scale2(v + 2, inv);
    return cvt_e4m3x2(a.x, a.y) | (cvt_e4m3x2(b.x, b.y) << 16);
}
__device__ __forceinline__ uint32_t cvt_e2m1x8(const float* v, float inv) {
    const float2 a = scale2(v, inv), b = scale2(v + 2, inv), c = scale2(v + 4, inv), d = scale2(v + 6, inv);
    uint32_t w;
    asm("{\n\t.reg .b8 p, q, r, s;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 p, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 q, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 r, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 s, %8, %7;\n\t"
        "mov.b32 %0, {p, q, r, s};\n\t}"
        : "=r"(w)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y), "f"(d.x), "f"(d.y));
    return w;
}

__device__ __forceinline__ float2 e4m3x2_to_f(uint32_t w) {
    return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w), __NV_E4M3)));
}
__device__ __forceinline__ float2 e2m1x2_to_f(uint32_t w) {
    return __half22float2(__half2(__nv_cvt_fp4x2_to_halfraw2(static_cast<__nv_fp4x2_storage_t>(w), __NV_E2M1)));
}

// Value of a stored scale byte.
template <MxFormat F>
__device__ __forceinline__ float scale_value(uint32_t byte) {
    if constexpr (Traits<F>::kPow2) {
        if (byte == 0xff) return __uint_as_float(0x7fc00000u);
        return byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);   // 0: 2^-127, a subnormal
    } else {
        return __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
    }
}

// Scale of a whole tensor (nvfp4) from its largest finite magnitude, times 1 / (6 * 448) rounded to fp32: puts the
// largest block scale at 448.  An infinity or NaN has its block's scale to itself and does not move the others' grid.
// 2^-100 keeps 1 / (s g) finite; a tensor with nothing finite but zeros keeps g = 1.
__device__ __forceinline__ float tensor_scale(uint32_t amax_bits) {
    const float a = __uint_as_float(amax_bits);
    if (amax_bits == 0) return 1.0f;
    return fmaxf(a * (1.0f / 2688.0f), 7.888609052210118e-31f);
}

// Overlap of a kernel's start with the end of the one before it (programmatic dependent launch).  allow_next lets the
// next kernel's CTAs start where there is room; wait_previous, before anything that another kernel may have written
// is read and before anything is written, waits until all that was launched before is complete.
// Measured back to back in a graph, without and with it: nvfp4 product of 1 x 4096 x 4096 7.6 and 6.0 us, norm to mxfp8
// of 10400 x 384 7.95 and 7.5, mxfp4 quantisation of 1536 x 384 3.2 and 2.6.
__device__ __forceinline__ void allow_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// ---------------------------------------------------------------- 16-byte vectors of the three input types
template <typename T>
struct VecOf {
    static constexpr int kN = 16 / sizeof(T);
};
__device__ __forceinline__ void unpack16(const uint4& w, float* f, __nv_bfloat16) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f[2 * i] = __uint_as_float(u[i] << 16);
        f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
}
__device__ __forceinline__ void unpack16(const uint4& w, float* f, __half) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        f[2 * i] = t.x;
        f[2 * i + 1] = t.y;
    }
}
__device__ __forceinline__ void unpack16(const uint4& w, float* f, float) {
    f[0] = __uint_as_float(w.x);
    f[1] = __uint_as_float(w.y);
    f[2] = __uint_as_float(w.z);
    f[3] = __uint_as_float(w.w);
}
__device__ __forceinline__ uint4 pack16(const float* f, __nv_bfloat16) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                      pack_bf16x2(f[6], f[7]));
}
__device__ __forceinline__ uint32_t pack_f16x2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint4 pack16(const float* f, __half) {
    return make_uint4(pack_f16x2(f[0], f[1]), pack_f16x2(f[2], f[3]), pack_f16x2(f[4], f[5]),
                      pack_f16x2(f[6], f[7]));
}
__device__ __forceinline__ uint4 pack16(const float* f, float) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}

__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ void ld_global_32(const void* p, uint4* w) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(w[0].x), "=r"(w[0].y), "=r"(w[0].z), "=r"(w[0].w), "=r"(w[1].x), "=r"(w[1].y), "=r"(w[1].z), "=r"(w[1].w)
                 : "l"(p));
}
__device__ __forceinline__ void st_global_32(void* p, const uint4& a, const uint4& b) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z),
                 "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
                 : "memory");
}

// ---------------------------------------------------------------- vectors at any element's address
// Bytes sh .. sh + 15 of the 32 in a, b.
__device__ __forceinline__ uint4 shift16(const uint4& a, const uint4& b, uint32_t sh) {
    uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    if (sh & 8) {
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (sh & 4) {
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    const uint32_t bits = (sh & 3) * 8;
    return make_uint4(__funnelshift_r(w[0], w[1], bits), __funnelshift_r(w[1], w[2], bits),
                      __funnelshift_r(w[2], w[3], bits), __funnelshift_r(w[3], w[4], bits));
}
// The 16 bytes of elements at p, of which the first n are read and the rest zero (n <= 0: none).  One or two aligned
// loads of 16-byte granules that hold at least one of the n, so nothing outside the allocation's granules is read.
template <typename T>
__device__ __forceinline__ uint4 load_any(const T* p, int n) {
    constexpr int kN = 16 / sizeof(T);
    if (n <= 0) return make_uint4(0, 0, 0, 0);
    const uintptr_t at = reinterpret_cast<uintptr_t>(p), base = at & ~uintptr_t(15);
    const uint32_t sh = static_cast<uint32_t>(at & 15);
    const uint4 a = *reinterpret_cast<const uint4*>(base);
    uint4 w = a;
    if (sh) {
        uint4 b = make_uint4(0, 0, 0, 0);
        if (base + 16 < at + n * sizeof(T)) b = *reinterpret_cast<const uint4*>(base + 16);
        w = shift16(a, b, sh);
    }
    if (n < kN) {      // zero the rest
        uint32_t* u = &w.x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int have = (n * static_cast<int>(sizeof(T)) - 4 * i) * 8;      // valid bits of this word
            u[i] = have >= 32 ? u[i] : (have <= 0 ? 0u : u[i] & (0xffffffffu >> (32 - have)));
        }
    }
    return w;
}
// Bytes from .. to - 1 of w (multiples of the element size) at p + from, where p + from or p + to is 16-byte aligned:
// pieces of 2, 4 and 8 bytes, rising from an unaligned start or falling from an aligned one.
__device__ __forceinline__ void store_part(char* p, const uint4& w, uint32_t from, uint32_t to) {
    const bool rising = (reinterpret_cast<uintptr_t>(p + from) & 15) != 0;
    const uint32_t count = to - from;
    uint32_t at = from;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        const uint32_t size = rising ? 2u << k : 8u >> k;
        if (count & size) {
            const uint4 v = shift16(w, make_uint4(0, 0, 0, 0), at);
            if (size == 2) *reinterpret_cast<unsigned short*>(p + at) = static_cast<unsigned short>(v.x);
            else if (size == 4) *reinterpret_cast<uint32_t*>(p + at) = v.x;
            else *reinterpret_cast<uint2*>(p + at) = make_uint2(v.x, v.y);
            at += size;
        }
    }
}
// Stores the first n elements of w at p, in the widest pieces that p's address allows.
template <typename T>
__device__ __forceinline__ void store_any_vec(T* p, const uint4& w, int n) {
    constexpr int kN = 16 / sizeof(T);
    const uint32_t sh = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) & 15);
    if (n >= kN && sh == 0) {
        *reinterpret_cast<uint4*>(p) = w;
    } else if (n >= kN && (sh & 7) == 0) {
        reinterpret_cast<uint2*>(p)[0] = make_uint2(w.x, w.y);
        reinterpret_cast<uint2*>(p)[1] = make_uint2(w.z, w.w);
    } else if (n >= kN && (sh & 3) == 0) {
        uint32_t* q = reinterpret_cast<uint32_t*>(p);
        q[0] = w.x;
        q[1] = w.y;
        q[2] = w.z;
        q[3] = w.w;
    } else if (n >= kN) {      // 16-bit elements at an odd one: half a word, three words, half a word
        unsigned short* h = reinterpret_cast<unsigned short*>(p);
        uint32_t* q = reinterpret_cast<uint32_t*>(h + 1);
        h[0] = static_cast<unsigned short>(w.x);
        q[0] = __funnelshift_r(w.x, w.y, 16);
        q[1] = __funnelshift_r(w.y, w.z, 16);
        q[2] = __funnelshift_r(w.z, w.w, 16);
        h[7] = static_cast<unsigned short>(w.w >> 16);
    } else {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < kN; ++i)
            if (i < n) {
                if constexpr (sizeof(T) == 4) reinterpret_cast<uint32_t*>(p)[i] = u[i];
                else reinterpret_cast<unsigned short*>(p)[i] = static_cast<unsigned short>(u[i >> 1] >> (16 * (i & 1)));
            }
    }
}

// Launch of a kernel that calls wait_previous.
template <typename... Params, typename... Args>
cudaError_t launch_early(void (*kern)(Params...), dim3 grid, int threads, cudaStream_t st, int smem, Args... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, static_cast<Params>(args)...);
}

// Lets a kernel use `bytes` of dynamic shared memory; asked of each device once (a launch's host time counts).
template <typename Kern>
cudaError_t allow_smem(Kern kern, std::atomic<uint64_t>& done, int bytes) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = uint64_t(1) << (dev & 63);
    if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) done.fetch_or(bit);
    return e;
}

inline int row_align(const void* p, int64_t pitch_bytes) {
    const uint64_t a = reinterpret_cast<uintptr_t>(p) | static_cast<uint64_t>(pitch_bytes);
    return a % 32 == 0 ? 2 : (a % 16 == 0 ? 1 : 0);
}

// 16 consecutive elements of a row as they are stored; elements at or past dim are zeros.
// align: the row starts at a multiple of 32 (2), of 16 (1) or of fewer bytes (0).
template <typename T>
struct Raw16 {
    static constexpr int kVecs = static_cast<int>(sizeof(T));
    uint4 w[kVecs];
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) w[i] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void load(const T* x, int64_t col, int64_t dim, int align) {
        if (align == 2 && col + 16 <= dim) {
#pragma unroll
            for (int i = 0; i < kVecs; i += 2) ld_global_32(reinterpret_cast<const uint4*>(x + col) + i, w + i);
        } else if (align && col + 16 <= dim) {
#pragma unroll
            for (int i = 0; i < kVecs; ++i) w[i] = reinterpret_cast<const uint4*>(x + col)[i];
        } else {
            const int n = static_cast<int>(dim - col < 16 ? dim - col : 16);
#pragma unroll
            for (int i = 0; i < kVecs; ++i) w[i] = load_any(x + col + i * VecOf<T>::kN, n - i * VecOf<T>::kN);
        }
    }
    __device__ __forceinline__ void get(float* v) const {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) unpack16(w[i], v + i * VecOf<T>::kN, T());
    }
    // largest magnitude, as fp32 bits; keeps a NaN (as integers, 16-bit magnitudes order like their values)
    __device__ __forceinline__ uint32_t amax_bits() const {
        if constexpr (sizeof(T) == 2) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < kVecs; ++i)
                m = max_u16x2(max_u16x2(max_u16x2(m, w[i].x & 0x7fff7fffu), w[i].y & 0x7fff7fffu),
                              max_u16x2(w[i].z & 0x7fff7fffu, w[i].w & 0x7fff7fffu));
            m = max(m & 0xffffu, m >> 16);
            if constexpr (std::is_same_v<T, __half>) return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(m))));
            return m << 16;
        } else {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < kVecs; ++i)
                m = max(max(max(m, w[i].x & 0x7fffffffu), w[i].y & 0x7fffffffu), max(w[i].z & 0x7fffffffu, w[i].w & 0x7fffffffu));
            return m;
        }
    }
};

}  // namespace mx
}  // namespace mmltk

// element type dispatch of the microscale / RMS-norm kernels (bf16, f16, fp32)
#define MMLTK_DISPATCH_ELT(et, ...)                    \
    [&]() -> cudaError_t {                             \
        if ((et) == ::mmltk::Elt::kBF16) {             \
            using elt_t = __nv_bfloat16;               \
            return __VA_ARGS__();                      \
        } else if ((et) == ::mmltk::Elt::kF16) {       \
            using elt_t = __half;                      \
            return __VA_ARGS__();                      \
        } else if ((et) == ::mmltk::Elt::kF32) {       \
            using elt_t = float;                       \
            return __VA_ARGS__();                      \
        }                                              \
        return cudaErrorInvalidValue;                  \
    }()
