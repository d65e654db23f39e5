// Quantisation to the microscaled formats (microscale.cuh), and back.
//
//   s = scale of a block from its largest magnitude, q = round(x / s) to the element type, value = q s (g)
//
// Memory-bound: 2 bytes in and 0.53 (4-bit) or 1.03 (8-bit) bytes out per 16-bit element.
// One CTA takes 128 rows x 128 elements, the rows of one scale tile: a thread holds 16 consecutive
// elements of each of the four rows r, r + 32, r + 64, r + 96, whose loads are all in flight together,
// and whose scale bytes are neighbours in the tile.  The tile is put together in shared memory and
// leaves in 16-byte stores; a tile built from byte stores of CTAs that run at different times would
// reach DRAM in parts.
#include "microscale.cuh"

namespace mmltk {

namespace {

using namespace mx;

constexpr int kTileRows = 128, kTileCols = 128;
constexpr int kQThreads = 256;

// 16 elements at x + col (col a multiple of 16); elements at or past dim read as zero.
template <typename T>
__device__ __forceinline__ void load16(const T* x, int64_t col, int64_t dim, bool vec, float* v) {
    if (vec && col + 16 <= dim) {
        constexpr int kN = VecOf<T>::kN;
#pragma unroll
        for (int i = 0; i < 16 / kN; ++i) unpack16(reinterpret_cast<const uint4*>(x + col)[i], v + i * kN, T());
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = col + i < dim ? to_f(x[col + i]) : 0.f;
    }
}

template <typename T, MxFormat F>
__global__ void __launch_bounds__(kQThreads) mx_quantize_kernel(const T* __restrict__ x, int64_t ld, int64_t rows,
                                                                int64_t dim, uint8_t* __restrict__ codes,
                                                                int64_t pitch, uint8_t* __restrict__ scales, int kt,
                                                                int64_t col_tiles, float* __restrict__ g_io,
                                                                const uint32_t* __restrict__ amax, bool vec) {
    using Tr = Traits<F>;
    constexpr int kAtoms = kTileCols / (4 * Tr::kBlock);     // scale tiles of this CTA: 1 or 2
    __shared__ __align__(16) uint8_t tile[kAtoms * 512];
    allow_next();
    // with amax the maximum was found by a pass in ascending order just before: going backwards, this pass
    // finds the end of x still in L2 (16384 x 8192 bf16)
    const int64_t unit = amax ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
    const int64_t rt = unit / col_tiles, ct = unit % col_tiles;
    float g = 1.f;
    if constexpr (!Tr::kPow2) {
        if (amax) {
            g = tensor_scale(*amax);
            if (unit == 0 && threadIdx.x == 0) *g_io = g;
        } else if (g_io) {
            g = *g_io;
        }
    }
    const int r32 = threadIdx.x >> 3, part = threadIdx.x & 7;
    const int64_t col = ct * kTileCols + part * 16;
    float v[4][16];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        const int64_t r = rt * kTileRows + 32 * s + r32;
        if (r < rows) {
            load16(x + r * ld, col, dim, vec, v[s]);
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) v[s][i] = 0.f;
        }
    }
    const int64_t pitch_cols = Tr::kBits == 4 ? 2 * pitch : pitch;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) m = max(m, abs_bits(v[s][i]));
        if constexpr (Tr::kBlock == 32) m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
        const BlockScale sc = block_scale<F>(__uint_as_float(m), g);
        const int64_t r = rt * kTileRows + 32 * s + r32;
        if (r < rows && col < pitch_cols) {
            if constexpr (Tr::kBits == 4) {
                *reinterpret_cast<uint2*>(codes + r * pitch + col / 2) =
                    make_uint2(cvt_e2m1x8(v[s], sc.inv), cvt_e2m1x8(v[s] + 8, sc.inv));
            } else {
                *reinterpret_cast<uint4*>(codes + r * pitch + col) =
                    make_uint4(cvt_e4m3x4(v[s], sc.inv), cvt_e4m3x4(v[s] + 4, sc.inv), cvt_e4m3x4(v[s] + 8, sc.inv),
                               cvt_e4m3x4(v[s] + 12, sc.inv));
            }
        }
        if constexpr (Tr::kBlock == 32) {
            if ((part & 1) == 0) tile[r32 * 16 + s * 4 + (part >> 1)] = static_cast<uint8_t>(sc.byte);
        } else {
            tile[(part >> 2) * 512 + r32 * 16 + s * 4 + (part & 3)] = static_cast<uint8_t>(sc.byte);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kAtoms * 32; i += kQThreads) {
        const int64_t atom = ct * kAtoms + i / 32;
        if (atom < kt)
            reinterpret_cast<uint4*>(scales + (rt * kt + atom) * 512)[i % 32] = reinterpret_cast<const uint4*>(tile)[i];
    }
}

// largest magnitude of a matrix, as bits (an order that keeps NaN); max does not depend on the order
template <typename T>
__global__ void __launch_bounds__(512) mx_amax_kernel(const T* __restrict__ x, int64_t ld, int64_t rows, int64_t dim,
                                                      uint32_t* __restrict__ amax, bool vec) {
    constexpr int kN = VecOf<T>::kN;
    uint32_t m = 0;
    if (vec) {   // whole 16-byte vectors: pitch, base and width all multiples
        const int64_t per_row = dim / kN, total = rows * per_row;
        const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
        int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
        const bool dense = ld == dim;
        for (; i + 3 * step < total; i += 4 * step) {
            uint4 w[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int64_t j = i + u * step;
                w[u] = dense ? reinterpret_cast<const uint4*>(x)[j]
                             : reinterpret_cast<const uint4*>(x + (j / per_row) * ld)[j % per_row];
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                float f[kN];
                unpack16(w[u], f, T());
#pragma unroll
                for (int e = 0; e < kN; ++e) m = max(m, abs_bits(f[e]));
            }
        }
        for (; i < total; i += step) {
            float f[kN];
            unpack16(reinterpret_cast<const uint4*>(x + (i / per_row) * ld)[i % per_row], f, T());
#pragma unroll
            for (int e = 0; e < kN; ++e) m = max(m, abs_bits(f[e]));
        }
    } else {
        const int64_t total = rows * dim;
        for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
             i += static_cast<int64_t>(gridDim.x) * blockDim.x)
            m = max(m, abs_bits(to_f(x[(i / dim) * ld + i % dim])));
    }
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0 && m) atomicMax(amax, m);
}

template <typename T, MxFormat F>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(const uint8_t* __restrict__ codes, int64_t pitch,
                                                            const uint8_t* __restrict__ scales, int kt,
                                                            const float* __restrict__ g_in, int64_t rows, int64_t dim,
                                                            T* __restrict__ out, bool vec) {
    using Tr = Traits<F>;
    const int64_t parts = (dim + 15) / 16;
    const float g = (!Tr::kPow2 && g_in) ? *g_in : 1.f;
    const int64_t total = rows * parts;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int64_t r = i / parts, col = (i % parts) * 16;
        const float s = scale_value<F>(scales[scale_offset(r, static_cast<int>(col / Tr::kBlock), kt)]);
        float v[16];
        if constexpr (Tr::kBits == 4) {
            const uint2 w = *reinterpret_cast<const uint2*>(codes + r * pitch + col / 2);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float2 t = e2m1x2_to_f(((e < 4 ? w.x : w.y) >> (8 * (e & 3))) & 0xff);
                v[2 * e] = t.x;
                v[2 * e + 1] = t.y;
            }
        } else {
            const uint4 w = *reinterpret_cast<const uint4*>(codes + r * pitch + col);
            const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float2 t = e4m3x2_to_f((u[e >> 1] >> (16 * (e & 1))) & 0xffff);
                v[2 * e] = t.x;
                v[2 * e + 1] = t.y;
            }
        }
        // (q s) is exact in fp32; the tensor's scale rounds once before the stored type does
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = v[e] * s * g;
        T* o = out + r * dim + col;
        if (vec && col + 16 <= dim) {
            constexpr int kN = VecOf<T>::kN;
#pragma unroll
            for (int e = 0; e < 16 / kN; ++e) reinterpret_cast<uint4*>(o)[e] = pack16(v + e * kN, T());
        } else {
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (col + e < dim) o[e] = from_f<T>(v[e]);
        }
    }
}

template <typename Fn>
cudaError_t by_format(MxFormat f, Fn&& fn) {
    if (f == MxFormat::kMxFp4) return fn(std::integral_constant<MxFormat, MxFormat::kMxFp4>{});
    if (f == MxFormat::kNvFp4) return fn(std::integral_constant<MxFormat, MxFormat::kNvFp4>{});
    return fn(std::integral_constant<MxFormat, MxFormat::kMxFp8>{});
}

}  // namespace

cudaError_t launch_mx_quantize(Elt et, MxFormat f, const void* x, int64_t ld, int64_t rows, int64_t dim, void* codes,
                               void* scales, float* g, uint32_t* amax, cudaStream_t st) {
    if (rows <= 0 || dim <= 0) return cudaSuccess;
    const int64_t row_tiles = (rows + kTileRows - 1) / kTileRows, col_tiles = (dim + kTileCols - 1) / kTileCols;
    if (row_tiles * col_tiles >= (int64_t(1) << 31)) return cudaErrorInvalidValue;
    return MMLTK_DISPATCH_ELT(et, [&]() -> cudaError_t {
        using T = elt_t;
        const int kN = 16 / static_cast<int>(sizeof(T));
        const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && ld % kN == 0;
        if (f == MxFormat::kNvFp4 && amax) {
            cudaError_t e = cudaMemsetAsync(amax, 0, sizeof(uint32_t), st);
            if (e != cudaSuccess) return e;
            const int64_t work = (rows * dim + 512 * kN * 4 - 1) / (512 * kN * 4);
            const int blocks = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(work, num_sms() * 4)));
            mx_amax_kernel<T><<<blocks, 512, 0, st>>>(static_cast<const T*>(x), ld, rows, dim, amax,
                                                      vec && dim % kN == 0);
            e = cudaGetLastError();
            if (e != cudaSuccess) return e;
        }
        return by_format(f, [&](auto fc) -> cudaError_t {
            constexpr MxFormat F = decltype(fc)::value;
            mx_quantize_kernel<T, F><<<static_cast<unsigned>(row_tiles * col_tiles), kQThreads, 0, st>>>(
                static_cast<const T*>(x), ld, rows, dim, static_cast<uint8_t*>(codes), mx_pitch(f, dim),
                static_cast<uint8_t*>(scales), static_cast<int>(mx_scale_tiles(f, dim)), col_tiles, g,
                F == MxFormat::kNvFp4 ? amax : nullptr, vec);
            return cudaGetLastError();
        });
    });
}

cudaError_t launch_mx_dequantize(Elt et, MxFormat f, const void* codes, const void* scales, const float* g,
                                 int64_t rows, int64_t dim, void* out, cudaStream_t st) {
    if (rows <= 0 || dim <= 0) return cudaSuccess;
    const int64_t total = rows * ((dim + 15) / 16);
    const int blocks = static_cast<int>(std::min<int64_t>((total + 255) / 256, static_cast<int64_t>(num_sms()) * 64));
    return MMLTK_DISPATCH_ELT(et, [&]() -> cudaError_t {
        using T = elt_t;
        const bool vec = reinterpret_cast<uintptr_t>(out) % 16 == 0 && dim % (16 / static_cast<int>(sizeof(T))) == 0;
        return by_format(f, [&](auto fc) -> cudaError_t {
            constexpr MxFormat F = decltype(fc)::value;
            mx_dequantize_kernel<T, F><<<blocks, 256, 0, st>>>(
                static_cast<const uint8_t*>(codes), mx_pitch(f, dim), static_cast<const uint8_t*>(scales),
                static_cast<int>(mx_scale_tiles(f, dim)), g, rows, dim, static_cast<T*>(out), vec);
            return cudaGetLastError();
        });
    });
}

}  // namespace mmltk
