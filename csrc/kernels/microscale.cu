// Quantisation to the microscaled formats (microscale.cuh), and back.
//
//   s = scale of a block from its largest magnitude, q = round(x / s) to the element type, value = q s (g)
//
// Memory-bound: 2 bytes in and 0.53 (4-bit) or 1.03 (8-bit) bytes out per 16-bit element.
// A thread takes 16 consecutive elements (one 32-byte load) of each of the four rows r, r + 32, r + 64,
// r + 96: the four loads are in flight together, held as loaded, and the four rows' scale bytes are
// neighbours in their tile.  The tiles' rows are put together in shared memory and leave as whole
// sectors; a tile built from byte stores of CTAs that run at different times would reach DRAM in parts.
// Measured, graph replays, 16384 x 8192 bf16: mxfp4 52 us (6.5 TB/s), nvfp4 54 us, with the tensor's scale found first
// 97 us (105 where replays alternate between two inputs: the end of x then waits in L2 for the second pass only), mxfp8
// 60 us; back to bf16 64 to 69 us (5.2 to 5.9 TB/s).  fp32: mxfp4 89 us, nvfp4 93 (105 at three CTAs an SM, which
// spill), mxfp8 97.  1536 x 384: 2.6 us, nvfp4 with its scale found 5.3.  Rows that are no multiple of 16 bytes
// (16384 x 8191): mxfp4 89 us, nvfp4 92 and 141, mxfp8 94; back 151 to 155 us: their loads and stores are cut at the
// granules of memory, vector by vector.  Reading all but the end of x past L2 in the pass for the scale (for the second
// pass to find more there) changed nothing: 97 and 97 us.
#include "microscale.cuh"

namespace mmltk {

namespace {

using namespace mx;

constexpr int kQThreads = 256, kAmaxThreads = 1024;

// kRow threads side by side in a row (8 or 32: 128 or 512 columns a CTA, of 4 x 32 or 4 x 8 rows).
template <typename T, MxFormat F, int kRow>
__global__ void __launch_bounds__(kQThreads, sizeof(T) == 2 ? 4 : 2)
    mx_quantize_kernel(const T* __restrict__ x, int64_t ld, int64_t rows, int64_t dim, uint8_t* __restrict__ codes,
                       int64_t pitch, uint8_t* __restrict__ scales, int kt, int col_tiles, int units,
                       float* __restrict__ g_io, const uint32_t* __restrict__ amax, int parts, int align) {
    using Tr = Traits<F>;
    constexpr int kCols = 16 * kRow, kLines = kQThreads / kRow;      // kLines: values of r % 32
    constexpr int kAtoms = kCols / (4 * Tr::kBlock);                 // scale tiles across a CTA's columns
    __shared__ __align__(16) uint8_t tile[kAtoms * kLines * 16];
    __shared__ uint32_t warp_max[kQThreads / 32];
    allow_next();
    wait_previous();
    // with amax the maximum was found by a pass in ascending order just before: going backwards, this pass
    // finds the end of x still in L2
    const int unit = amax ? units - 1 - static_cast<int>(blockIdx.x) : static_cast<int>(blockIdx.x);
    const int ct = unit % col_tiles, line = unit / col_tiles;
    float g = 1.f;
    if constexpr (!Tr::kPow2) {
        if (!amax && g_io) g = *g_io;
    }
    const int l = threadIdx.x / kRow, part = threadIdx.x % kRow;
    const int64_t rt = static_cast<int64_t>(line) / (32 / kLines);
    const int r32 = line % (32 / kLines) * kLines + l;
    const int64_t r0 = rt * 128 + r32, col = static_cast<int64_t>(ct) * kCols + part * 16;
    Raw16<T> raw[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        if (r0 + 32 * s < rows && col < dim) raw[s].load(x + (r0 + 32 * s) * ld, col, dim, align);
        else raw[s].zero();
    }
    if constexpr (!Tr::kPow2) {
        if (amax) {
            uint32_t m = 0;
            for (int i = threadIdx.x; i < parts; i += kQThreads) m = max(m, amax[i]);
            m = __reduce_max_sync(0xffffffffu, m);
            if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kQThreads / 32; ++i) m = max(m, warp_max[i]);
            g = tensor_scale(m);
            if (unit == 0 && threadIdx.x == 0) *g_io = g;
        }
    }
    const int64_t pitch_cols = Tr::kBits == 4 ? 2 * pitch : pitch;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
        uint32_t m = raw[s].amax_bits();
        if constexpr (Tr::kBlock == 32) m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
        const BlockScale sc = block_scale<F>(__uint_as_float(m), g);
        const int64_t r = r0 + 32 * s;
        float v[16];
        raw[s].get(v);
        if (r < rows && col < pitch_cols) {
            if constexpr (Tr::kBits == 4) {
                *reinterpret_cast<uint2*>(codes + r * pitch + col / 2) =
                    make_uint2(cvt_e2m1x8(v, sc.inv), cvt_e2m1x8(v + 8, sc.inv));
            } else {
                *reinterpret_cast<uint4*>(codes + r * pitch + col) =
                    make_uint4(cvt_e4m3x4(v, sc.inv), cvt_e4m3x4(v + 4, sc.inv), cvt_e4m3x4(v + 8, sc.inv),
                               cvt_e4m3x4(v + 12, sc.inv));
            }
        }
        if constexpr (Tr::kBlock == 32) {
            if ((part & 1) == 0) tile[((part >> 3) * kLines + l) * 16 + s * 4 + ((part >> 1) & 3)] = static_cast<uint8_t>(sc.byte);
        } else {
            tile[((part >> 2) * kLines + l) * 16 + s * 4 + (part & 3)] = static_cast<uint8_t>(sc.byte);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < kAtoms * kLines; i += kQThreads) {
        const int atom = ct * kAtoms + i / kLines;
        if (atom < kt)
            reinterpret_cast<uint4*>(scales + (rt * kt + atom) * 512)[line % (32 / kLines) * kLines + i % kLines] =
                reinterpret_cast<const uint4*>(tile)[i];
    }
}

// Running largest finite magnitude.  A magnitude's bits plus the distance from infinity to the sign bit stay positive, in
// order, for finite numbers and turn negative for infinities and NaN, which a signed maximum then passes over: one
// instruction a word beside the mask.
template <typename T>
struct FiniteMax {
    static constexpr bool kWide = sizeof(T) == 4;
    static constexpr uint32_t kOne = kWide ? 0x00800000u : (std::is_same_v<T, __half> ? 0x0400u : 0x0080u);
    static constexpr uint32_t kBias = kWide ? kOne : kOne | kOne << 16;
    uint32_t m = kBias;
    __device__ __forceinline__ void word(uint32_t w) {
        if constexpr (kWide) m = static_cast<uint32_t>(__viaddmax_s32(static_cast<int>(w & 0x7fffffffu), static_cast<int>(kBias), static_cast<int>(m)));
        else m = __viaddmax_s16x2(w & 0x7fff7fffu, kBias, m);
    }
    __device__ __forceinline__ void add(const uint4& w) {
        word(w.x);
        word(w.y);
        word(w.z);
        word(w.w);
    }
    __device__ __forceinline__ uint32_t bits() const {      // of the value as fp32
        if constexpr (kWide) return m - kOne;
        const uint32_t t = max(m & 0xffffu, m >> 16) - kOne;
        if constexpr (std::is_same_v<T, __half>) return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(t))));
        return t << 16;
    }
};

// Largest finite magnitude of each CTA's part of a matrix, as bits (max does not depend on the order); the pass that
// reads them takes the largest.  A dense matrix is read as one row.
template <typename T>
__global__ void __launch_bounds__(kAmaxThreads) mx_amax_kernel(const T* __restrict__ x, int64_t ld, int64_t rows, int64_t dim,
                                                      uint32_t* __restrict__ amax) {
    constexpr int kN = VecOf<T>::kN;
    __shared__ uint32_t warp_max[kAmaxThreads / 32];
    FiniteMax<T> top;
    wait_previous();
    // CTAs side by side in a row, then over the rows
    const int64_t step = static_cast<int64_t>(gridDim.x) * blockDim.x;
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
        const T* row = x + r * ld;
        int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
        const bool aligned = reinterpret_cast<uintptr_t>(row) % 16 == 0;
        const int64_t whole = aligned ? dim / kN : 0, total = (dim + kN - 1) / kN;
        for (; i + 3 * step < whole; i += 4 * step) {
            uint4 w[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) w[u] = reinterpret_cast<const uint4*>(row)[i + u * step];
#pragma unroll
            for (int u = 0; u < 4; ++u) top.add(w[u]);
        }
        for (; i < total; i += step) {
            const int64_t left = dim - i * kN;
            top.add(load_any(row + i * kN, left < kN ? static_cast<int>(left) : kN));
        }
    }
    allow_next();
    uint32_t m = __reduce_max_sync(0xffffffffu, top.bits());
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
    __syncthreads();
    if (threadIdx.x >= 32) return;
    m = threadIdx.x < kAmaxThreads / 32 ? warp_max[threadIdx.x] : 0;
    m = __reduce_max_sync(0xffffffffu, m);
    if (threadIdx.x == 0) amax[blockIdx.y * gridDim.x + blockIdx.x] = m;
}

// 16 values of a lane to an unaligned place: the aligned granules between its vectors whole, the ends in pieces.
template <typename T>
__device__ __forceinline__ void lane_store(T* o, const float* v, int n) {
    constexpr int kN = VecOf<T>::kN;
    if (n < 16) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
            if (e < n) o[e] = from_f<T>(v[e]);
        return;
    }
    char* c = reinterpret_cast<char*>(o);
    const uint32_t head = (16 - static_cast<uint32_t>(reinterpret_cast<uintptr_t>(o) & 15)) & 15;
    uint4 w = pack16(v, T());
    if (head) store_part(c, w, 0, head);
#pragma unroll
    for (int e = kN; e < 16; e += kN) {
        const uint4 u = pack16(v + e, T());
        *reinterpret_cast<uint4*>(c + (e / kN - 1) * 16 + head) = head ? shift16(w, u, head) : w;
        w = u;
    }
    c += (16 / kN - 1) * 16;
    if (head) store_part(c, w, head, 16);
    else *reinterpret_cast<uint4*>(c) = w;
}

// A thread writes 16 consecutive values (one 32-byte store of a 16-bit type); a CTA's y is a row of
// CTAs, its x the columns.
template <typename T, MxFormat F, bool kWhole>     // kWhole: rows are 32-byte aligned
__global__ void __launch_bounds__(256) mx_dequantize_kernel(const uint8_t* __restrict__ codes, int64_t pitch,
                                                            const uint8_t* __restrict__ scales, int kt,
                                                            const float* __restrict__ g_in, int64_t rows, int64_t dim,
                                                            int parts, int part_bits, T* __restrict__ out) {
    using Tr = Traits<F>;
    const float g = (!Tr::kPow2 && g_in) ? *g_in : 1.f;
    // 2^part_bits threads side by side in a row
    const int part0 = threadIdx.x & ((1 << part_bits) - 1), line = threadIdx.x >> part_bits, lines = 256 >> part_bits;
    const int part = (blockIdx.x << part_bits) + part0;
    for (int64_t r = static_cast<int64_t>(blockIdx.y) * lines + line; r < rows; r += static_cast<int64_t>(gridDim.y) * lines) {
        const int64_t col = static_cast<int64_t>(part) * 16;
        if (part >= parts) continue;
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
        constexpr int kN = VecOf<T>::kN;
        if (kWhole && col + 16 <= dim) {
#pragma unroll
            for (int e = 0; e < 16; e += 2 * kN) st_global_32(o + e, pack16(v + e, T()), pack16(v + e + kN, T()));
        } else {
            lane_store<T>(o, v, static_cast<int>(dim - col < 16 ? dim - col : 16));
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
    // 512 columns a CTA where a row has them (rows' loads of 1 KB); 128 for narrow matrices, whose CTAs would idle
    const int row_threads = dim > 256 ? 32 : 8;
    const int64_t col_tiles = (dim + 16 * row_threads - 1) / (16 * row_threads);
    const int64_t units = (rows + 127) / 128 * (row_threads / 8) * col_tiles;
    if (units >= (int64_t(1) << 31)) return cudaErrorInvalidValue;
    return MMLTK_DISPATCH_ELT(et, [&]() -> cudaError_t {
        using T = elt_t;
        const int kN = 16 / static_cast<int>(sizeof(T));
        const int align = row_align(x, ld * static_cast<int64_t>(sizeof(T)));
        int parts = 0;
        if (f == MxFormat::kNvFp4 && amax) {
            const int64_t most = std::min<int64_t>(2 * num_sms(), kMxAmaxParts);
            const int64_t r = ld == dim ? 1 : rows, d = ld == dim ? rows * dim : dim;
            const int64_t across =
                std::max<int64_t>(1, std::min((d + kAmaxThreads * kN - 1) / (kAmaxThreads * kN), most));
            const dim3 grid(static_cast<unsigned>(across),
                            static_cast<unsigned>(std::min(r, std::max<int64_t>(1, most / across))));
            parts = static_cast<int>(grid.x * grid.y);
            const cudaError_t e = launch_early(mx_amax_kernel<T>, grid, kAmaxThreads, st, 0, static_cast<const T*>(x), ld, r,
                                               d, amax);
            if (e != cudaSuccess) return e;
        }
        return by_format(f, [&](auto fc) -> cudaError_t {
            constexpr MxFormat F = decltype(fc)::value;
            auto run = [&](auto kern) {
                return launch_early(kern, dim3(static_cast<unsigned>(units)), kQThreads, st, 0, static_cast<const T*>(x), ld,
                                    rows, dim, static_cast<uint8_t*>(codes), mx_pitch(f, dim),
                                    static_cast<uint8_t*>(scales), static_cast<int>(mx_scale_tiles(f, dim)),
                                    static_cast<int>(col_tiles), static_cast<int>(units), g,
                                    F == MxFormat::kNvFp4 ? amax : nullptr, parts, align);
            };
            if (row_threads == 32) return run(mx_quantize_kernel<T, F, 32>);
            return run(mx_quantize_kernel<T, F, 8>);
        });
    });
}

cudaError_t launch_mx_dequantize(Elt et, MxFormat f, const void* codes, const void* scales, const float* g,
                                 int64_t rows, int64_t dim, void* out, cudaStream_t st) {
    if (rows <= 0 || dim <= 0) return cudaSuccess;
    const int64_t parts = (dim + 15) / 16;
    if (parts >= (int64_t(1) << 30)) return cudaErrorInvalidValue;
    int bits = 0;
    while (bits < 8 && (int64_t(1) << bits) < parts) ++bits;
    const int64_t lines = 256 >> bits;
    const dim3 grid(static_cast<unsigned>((parts + (1 << bits) - 1) >> bits),
                    static_cast<unsigned>(std::min<int64_t>((rows + lines - 1) / lines, 65535)));
    return MMLTK_DISPATCH_ELT(et, [&]() -> cudaError_t {
        using T = elt_t;
        const int align = row_align(out, dim * static_cast<int64_t>(sizeof(T)));
        return by_format(f, [&](auto fc) -> cudaError_t {
            constexpr MxFormat F = decltype(fc)::value;
            auto run = [&](auto kern) {
                kern<<<grid, 256, 0, st>>>(static_cast<const uint8_t*>(codes), mx_pitch(f, dim),
                                           static_cast<const uint8_t*>(scales), static_cast<int>(mx_scale_tiles(f, dim)),
                                           g, rows, dim, static_cast<int>(parts), bits, static_cast<T*>(out));
                return cudaGetLastError();
            };
            if (align == 2) return run(mx_dequantize_kernel<T, F, true>);
            return run(mx_dequantize_kernel<T, F, false>);
        });
    });
}

}  // namespace mmltk
