// Root-mean-square norm over the last dimension, with the residual's addition, and its backward.
//
//   h = round(x + r),  rstd = (mean(h^2) + eps)^-1/2,  y = h rstd w
//   gx = gr = gh + rstd w gy - h rstd^3 mean(h w gy),   gw = sum_rows gy h rstd
//
// y goes out in x's type, or quantised (microscale.cuh) straight from its fp32 values, with the
// scales in the tiled layout that the tensor-core product reads.
//
// Memory-bound.  A row is held in registers by a group of threads -- a warp up to 1024 16-bit
// elements, a CTA of 128 to 512 threads beyond -- so every element is read once; statistics are
// fp32.  A thread's elements are 16-byte vectors kGroup vectors apart, so the 2 to 8 threads of a
// scale block are neighbours in a warp and find its maximum with at most three shuffles.
// Measured, bf16 with a residual, graph replays: forward 32768 x 4096 157 us (6.8 TB/s), to mxfp8 139 us (6.8 TB/s), to
// mxfp4 136, to nvfp4 146; backward 160 us (6.7 TB/s); 16384 x 7001, whose rows start anywhere, 145 and 175 us (at the
// copy's rate 140 and 123), its backward without a residual 160 (105).  Replays write over outputs that are still in L2 as
// the last one left them, which saves some of their way to memory; single calls of 32768 x 4096 to mxfp8 with other
// buffers in between take 154 to 162 us.
#include "microscale.cuh"
#include "tcgen05.cuh"

namespace mmltk {

namespace {

using namespace mx;

constexpr int kRingStages = 8, kRingBytes = 216 * 1024;

// Where the rows start.  kWhole: every row on a 16-byte boundary.  kPhase: anywhere, but row r of every tensor equally far
// past one (dense tensors of any width): the vectors are then the aligned granules of a row, the first one reaching
// `lead` elements before it and the last one behind it, and only the weights have to be shifted.  kAny: each
// tensor in its own way; vectors start with the row, are read in aligned granules and shifted, and are written
// in the widest pieces the address allows.  bf16 with a residual, us as kAny and kPhase:
// 16384 x 7001 forward 261 and 145, to mxfp8 256 and 175, backward 263 and 162; 32768 x 518 42 and 38, 51 and 46, 76 and 69.
enum Rows { kWhole, kPhase, kAny };

// A vector of a row as loaded: unpacked where it is used, so that a waiting row takes 4 registers per 16 bytes
// (8 as fp32), which is what decides how many rows an SM has in flight.  i: its first element in the row (below 0 for
// kPhase's first one), below dim.  Elements outside the row read as zeros and are not written.
template <typename T, Rows kRows>
struct Raw {
    static constexpr int kN = VecOf<T>::kN;
    uint4 w;
    __device__ __forceinline__ void load(const T* row, int i, int dim) {
        if constexpr (kRows == kAny) {
            w = load_any(row + i, min(dim - i, kN));
        } else {
            w = *reinterpret_cast<const uint4*>(row + i);
        }
    }
    // kPhase: zeros outside the row; called when all of a row's loads have been issued, since it waits for one
    __device__ __forceinline__ void trim(int i, int dim) {
        if constexpr (kRows == kPhase) {
            if (i < 0 || i + kN > dim) {
                uint32_t* u = &w.x;
#pragma unroll
                for (int e = 0; e < kN; ++e)
                    if (i + e < 0 || i + e >= dim) {
                        if constexpr (sizeof(T) == 4) u[e] = 0;
                        else u[e / 2] &= e & 1 ? 0x0000ffffu : 0xffff0000u;
                    }
            }
        }
    }
    __device__ __forceinline__ void store(T* row, int i, int dim) const {
        if constexpr (kRows == kAny) {
            store_any_vec(row + i, w, min(dim - i, kN));
        } else if (kRows == kWhole || (i >= 0 && i + kN <= dim)) {
            *reinterpret_cast<uint4*>(row + i) = w;
        } else if (i >= 0 || i + kN <= dim) {
            constexpr int kSize = sizeof(T);
            store_part(reinterpret_cast<char*>(row + i), w, i < 0 ? -i * kSize : 0, min(kN, dim - i) * kSize);
        } else {      // a row inside one granule
            store_any_vec(row, shift16(w, make_uint4(0, 0, 0, 0), -i * static_cast<int>(sizeof(T))), dim);
        }
    }
    __device__ __forceinline__ void get(float* f) const { unpack16(w, f, T()); }
    __device__ __forceinline__ void set(const float* f) { w = pack16(f, T()); }
    __device__ __forceinline__ void zero() { w = make_uint4(0, 0, 0, 0); }
};

// Weights of x's type at any element i: the two granules, loaded, and shifted where they are used.  Elements outside the
// row are arbitrary.
template <typename T>
struct RawPair {
    uint4 a, b;
    __device__ __forceinline__ void load(const T* w, int i, int dim, int sh) {      // w + i is sh bytes past a granule
        const int at = i * static_cast<int>(sizeof(T)) - sh, end = dim * static_cast<int>(sizeof(T));
        const char* p = reinterpret_cast<const char*>(w) + at;
        a = at >= 0 && at < end ? *reinterpret_cast<const uint4*>(p) : make_uint4(0, 0, 0, 0);
        b = sh && at + 16 < end ? *reinterpret_cast<const uint4*>(p + 16) : make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void get(float* f, int sh) const { unpack16(shift16(a, b, sh), f, T()); }
};

// weights (16-byte aligned): x's type or fp32; zeros outside the row
template <typename T, Rows kRows>
__device__ __forceinline__ void load_w(const void* w, bool f32, int i, int dim, float* f) {
    constexpr int kN = VecOf<T>::kN;
    if (kRows != kWhole && (i < 0 || i + kN > dim)) {
#pragma unroll
        for (int e = 0; e < kN; ++e)
            f[e] = i + e < 0 || i + e >= dim ? 0.f
                   : f32                     ? static_cast<const float*>(w)[i + e]
                                             : to_f(static_cast<const T*>(w)[i + e]);
    } else if (f32) {
        const float* p = static_cast<const float*>(w) + i;
#pragma unroll
        for (int e = 0; e < kN; e += 4) {
            const uint4 t = kRows == kPhase ? load_any(p + e, 4) : *reinterpret_cast<const uint4*>(p + e);
            unpack16(t, f + e, float());
        }
    } else {
        const T* p = static_cast<const T*>(w) + i;
        unpack16(kRows == kPhase ? load_any(p, kN) : *reinterpret_cast<const uint4*>(p), f, T());
    }
}

// Sum over the kGroup threads of a row, the same value (and order) in all of them.
template <int kGroup>
__device__ __forceinline__ float group_sum(float s, float* red) {
    s = warp_sum(s);
    if constexpr (kGroup > 32) {
        constexpr int kWarps = kGroup / 32;
        const int lane = threadIdx.x & 31;
        if (lane == 0) red[threadIdx.x >> 5] = s;
        __syncthreads();
        s = warp_sum(lane < kWarps ? red[lane] : 0.f);
    }
    return s;
}

// Quantises the VEC values at column i of row r (a whole warp calls; i < span), stores codes and scales.
template <MxFormat F, int VEC>
__device__ __forceinline__ void quantize_store(const float* v, int i, int64_t r, int64_t pitch, int kt, int span,
                                               uint8_t* codes, uint8_t* scales, float g) {
    using Tr = Traits<F>;
    constexpr int kThreads = Tr::kBlock / VEC;      // threads of a block: 8 / 4 or 4 / 2
    static_assert(4 * kThreads <= 32);
    float top = 0.f;      // keeps a NaN
#pragma unroll
    for (int e = 0; e < VEC; e += 2) top = max3_abs_nan(top, v[e], v[e + 1]);
    uint32_t m = abs_bits(top);
#pragma unroll
    for (int o = 1; o < kThreads; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const BlockScale sc = block_scale<F>(__uint_as_float(m), g);
    const int lane = threadIdx.x & 31;
    uint8_t* row = codes + r * pitch;
    if constexpr (Tr::kBits == 8) {
        if (i < pitch) {
            if constexpr (VEC == 8)
                *reinterpret_cast<uint2*>(row + i) = make_uint2(cvt_e4m3x4(v, sc.inv), cvt_e4m3x4(v + 4, sc.inv));
            else
                *reinterpret_cast<uint32_t*>(row + i) = cvt_e4m3x4(v, sc.inv);
        }
    } else {
        if (i < 2 * pitch) {
            if constexpr (VEC == 8) {
                *reinterpret_cast<uint32_t*>(row + (i >> 1)) = cvt_e2m1x8(v, sc.inv);
            } else {
                const float2 a = scale2(v, sc.inv), b = scale2(v + 2, sc.inv);
                *reinterpret_cast<uint16_t*>(row + (i >> 1)) =
                    static_cast<uint16_t>(cvt_e2m1x2(a.x, a.y) | (cvt_e2m1x2(b.x, b.y) << 8));
            }
        }
    }
    // the four scales of a tile's row, one 4-byte store
    uint32_t b = sc.byte;
    b |= __shfl_down_sync(0xffffffffu, b, kThreads) << 8;
    b |= __shfl_down_sync(0xffffffffu, b, 2 * kThreads) << 16;
    if (i < span && (lane & (4 * kThreads - 1)) == 0)
        *reinterpret_cast<uint32_t*>(scales + scale_offset(r, i / Tr::kBlock, kt)) = b;
}

template <typename T, Rows kRows, int kGroup, int KV, bool kQuant>
__global__ void __launch_bounds__(kGroup == 32 ? 256 : kGroup,
                                  KV <= 4 ? 1024 / (kGroup == 32 ? 256 : kGroup) : 1)
    rms_fwd_kernel(RmsFwdArgs a) {
    constexpr int VEC = VecOf<T>::kN;
    __shared__ float red[32];
    extern __shared__ uint4 granules[];
    allow_next();
    wait_previous();
    constexpr int kPer = kGroup == 32 ? 8 : 1;
    const int64_t r = static_cast<int64_t>(blockIdx.x) * kPer + (kGroup == 32 ? threadIdx.x >> 5 : 0);
    const int t = kGroup == 32 ? threadIdx.x & 31 : threadIdx.x;
    const int kt = kQuant ? static_cast<int>(mx_scale_tiles(a.fmt, a.dim)) : 0;
    if (r >= a.rows) {   // (all of the row's threads) rows that fill the last scale tile: zero scales
        if (kQuant && r < (a.rows + 127) / 128 * 128)
            for (int i = t; i < kt; i += kGroup)
                *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(a.scales) + scale_offset(r, 4 * i, kt)) = 0;
        return;
    }
    [[maybe_unused]] uint4* buf = granules + (kGroup == 32 ? threadIdx.x >> 5 : 0) * KV * kGroup;
    const T* xr = static_cast<const T*>(a.x) + r * a.ldx;
    const T* rr = a.res ? static_cast<const T*>(a.res) + r * a.ldr : nullptr;
    const int lead = kRows == kPhase ? static_cast<int>(r * a.dim % VEC) : 0;
    Raw<T, kRows> v[KV];
#pragma unroll
    for (int k = 0; k < KV; ++k) {
        const int i = (k * kGroup + t) * VEC - lead;
        if (i < a.dim) v[k].load(xr, i, a.dim);
        else v[k].zero();
    }
    auto trim = [&](Raw<T, kRows>(&row)[KV]) {
        if constexpr (kRows == kPhase)
#pragma unroll
            for (int k = 0; k < KV; ++k) row[k].trim((k * kGroup + t) * VEC - lead, a.dim);
    };
    float s = 0.f;
    if (rr) {
        T* hr = static_cast<T*>(a.h) + r * a.dim;
        Raw<T, kRows> u[KV];
#pragma unroll
        for (int k = 0; k < KV; ++k) {
            const int i = (k * kGroup + t) * VEC - lead;
            if (i < a.dim) u[k].load(rr, i, a.dim);
            else u[k].zero();
        }
        trim(v);
        trim(u);
#pragma unroll
        for (int k = 0; k < KV; ++k) {
            const int i = (k * kGroup + t) * VEC - lead;
            if (i < a.dim) {
                // the norm sees the sum as it is stored, so that its backward can start from h
                float f[VEC], e[VEC];
                v[k].get(f);
                u[k].get(e);
#pragma unroll
                for (int j = 0; j < VEC; ++j) f[j] += e[j];
                v[k].set(f);
                v[k].store(hr, i, a.dim);
            }
        }
    } else {
        trim(v);
    }
#pragma unroll
    for (int k = 0; k < KV; ++k) {
        float f[VEC];
        v[k].get(f);
#pragma unroll
        for (int j = 0; j < VEC; ++j) s = fmaf(f[j], f[j], s);
    }
    if constexpr (kQuant && kRows == kPhase) {      // the blocks start with the row: the granules meet in shared memory
#pragma unroll
        for (int k = 0; k < KV; ++k) buf[k * kGroup + t] = v[k].w;
        if constexpr (kGroup == 32) __syncwarp();
    }
    s = group_sum<kGroup>(s, red);
    const float rstd = 1.f / sqrtf(s / static_cast<float>(a.dim) + a.eps);
    if (a.rstd && t == 0) a.rstd[r] = rstd;
    const int span = kQuant ? kt * 4 * mx_block(a.fmt) : a.dim;
    float g = 1.f;
    if (kQuant && a.g) g = *a.g;
    const int shift = kQuant ? 0 : lead;
    // kPhase: weights of x's type, two vectors' on their way before the first is shifted
    constexpr bool kPairs = kRows == kPhase && !kQuant;
    const bool pairs = kPairs && (sizeof(T) == 4 || !a.w_f32);
    const int wsh = lead ? 16 - lead * static_cast<int>(sizeof(T)) : 0;
    RawPair<T> wp[2];
#pragma unroll
    for (int k = 0; k < KV; ++k) {
        const int i = (k * kGroup + t) * VEC - shift;
        if (kPairs && pairs && k % 2 == 0) {
#pragma unroll
            for (int u = 0; u < (KV - k < 2 ? 1 : 2); ++u)
                wp[u].load(static_cast<const T*>(a.w), i + u * kGroup * VEC, a.dim, wsh);
        }
        if constexpr (kQuant && kRows == kPhase) {      // (after group_sum's barrier)
            const int j = k * kGroup + t;
            if (lead) v[k].w = shift16(buf[j], j + 1 < KV * kGroup ? buf[j + 1] : make_uint4(0, 0, 0, 0), lead * sizeof(T));
        }
        float f[VEC];
        v[k].get(f);
        if (i < a.dim) {
            float w[VEC];
            if (kPairs && pairs) wp[k % 2].get(w, wsh);
            else load_w<T, kQuant && kRows == kPhase ? kAny : kRows>(a.w, a.w_f32, i, a.dim, w);
#pragma unroll
            for (int j = 0; j < VEC; ++j) f[j] = f[j] * rstd * w[j];
            if constexpr (!kQuant) {
                Raw<T, kRows> y;
                y.set(f);
                y.store(static_cast<T*>(a.y) + r * a.dim, i, a.dim);
            }
        }
        if constexpr (kQuant) {
            if ((k * kGroup + (t & ~31)) * VEC >= span) continue;     // warp-uniform
            uint8_t* codes = static_cast<uint8_t*>(a.codes);
            uint8_t* scales = static_cast<uint8_t*>(a.scales);
            const int64_t pitch = mx_pitch(a.fmt, a.dim);
            if (a.fmt == MxFormat::kMxFp8)
                quantize_store<MxFormat::kMxFp8, VEC>(f, i, r, pitch, kt, span, codes, scales, g);
            else if (a.fmt == MxFormat::kMxFp4)
                quantize_store<MxFormat::kMxFp4, VEC>(f, i, r, pitch, kt, span, codes, scales, g);
            else
                quantize_store<MxFormat::kNvFp4, VEC>(f, i, r, pitch, kt, span, codes, scales, g);
        }
    }
}

// ---------------------------------------------------------------- backward
// Persistent: a group of threads walks rows and keeps its columns' part of gw in registers; one partial
// row per CTA, summed in a fixed order by rms_gw_kernel (no atomics: the same bits every run).
template <typename T, Rows kRows, int kGroup, int KV>
__global__ void __launch_bounds__(kGroup == 32 ? 256 : kGroup, kGroup == 32 ? 3 : 1) rms_bwd_kernel(RmsBwdArgs a) {
    constexpr int VEC = VecOf<T>::kN;
    constexpr int kPer = kGroup == 32 ? 8 : 1;
    __shared__ float red[2][32];
    __shared__ float part[kGroup == 32 ? 8 * 32 * VEC : 1];
    const int sub = kGroup == 32 ? threadIdx.x >> 5 : 0;
    const int t = threadIdx.x & (kGroup - 1);
    float acc[KV][VEC];
#pragma unroll
    for (int k = 0; k < KV; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[k][e] = 0.f;
    const float inv_dim = 1.f / static_cast<float>(a.dim);
    int turn = 0;
    for (int64_t r = static_cast<int64_t>(blockIdx.x) * kPer + sub; r < a.rows;
         r += static_cast<int64_t>(gridDim.x) * kPer, turn ^= 1) {
        const float rstd = a.rstd[r];
        Raw<T, kRows> hv[KV], gv[KV], ev[KV];
#pragma unroll
        for (int k = 0; k < KV; ++k) {
            const int i = (k * kGroup + t) * VEC;
            if (i < a.dim) {
                hv[k].load(static_cast<const T*>(a.h) + r * a.ldh, i, a.dim);
                gv[k].load(static_cast<const T*>(a.gy) + r * a.ldgy, i, a.dim);
                if (a.gh) ev[k].load(static_cast<const T*>(a.gh) + r * a.ldgh, i, a.dim);
            }
        }
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < KV; ++k) {
            const int i = (k * kGroup + t) * VEC;
            if (i < a.dim) {
                float w[VEC], h[VEC], g[VEC];
                load_w<T, kRows>(a.w, a.w_f32, i, a.dim, w);
                hv[k].get(h);
                gv[k].get(g);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    acc[k][e] = fmaf(g[e], h[e] * rstd, acc[k][e]);
                    s = fmaf(h[e], g[e] * w[e], s);
                }
            }
        }
        s = group_sum<kGroup>(s, red[turn]);     // two turns: the next row's sums do not meet this row's readers
        const float c = s * inv_dim * rstd * rstd * rstd;
#pragma unroll
        for (int k = 0; k < KV; ++k) {
            const int i = (k * kGroup + t) * VEC;
            if (i < a.dim) {
                float w[VEC], h[VEC], g[VEC];
                load_w<T, kRows>(a.w, a.w_f32, i, a.dim, w);
                hv[k].get(h);
                gv[k].get(g);
#pragma unroll
                for (int e = 0; e < VEC; ++e) g[e] = fmaf(rstd, g[e] * w[e], -c * h[e]);
                if (a.gh) {
                    ev[k].get(h);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) g[e] += h[e];
                }
                hv[k].set(g);
                hv[k].store(static_cast<T*>(a.gx) + r * a.dim, i, a.dim);
            }
        }
    }
    if (!a.partial) return;
    float* dst = a.partial + static_cast<int64_t>(blockIdx.x) * rms_partial_pitch(a.dim);
#pragma unroll
    for (int k = 0; k < KV; ++k) {
        const int i = (k * kGroup + t) * VEC;
        if constexpr (kGroup == 32) {
            // the eight warps' parts of these columns, added in the order of the warps
            __syncthreads();
#pragma unroll
            for (int e = 0; e < VEC; ++e) part[(sub * VEC + e) * 32 + t] = acc[k][e];
            __syncthreads();
            for (int j = threadIdx.x; j < 32 * VEC; j += 256) {
                const int lane = j / VEC, e = j % VEC, col = (k * 32 + lane) * VEC + e;
                float sum = 0.f;
#pragma unroll
                for (int w = 0; w < 8; ++w) sum += part[(w * VEC + e) * 32 + lane];
                if (col < a.dim) dst[col] = sum;
            }
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (i + e < a.dim) dst[i + e] = acc[k][e];
        }
    }
}

// The same for rows of more than a warp: the inputs come through a ring of rows in shared memory (bulk asynchronous
// copies), so what is in flight does not depend on registers; a row's stage is loaded again after the next row's
// sum, when every thread has left it.  bf16, us (TB/s; loads into registers): 16384 x 8192 167 (6.4; 197), 32768 x 4096
// 160 (6.7; 198), 65536 x 1024 97 (5.5; 119): a row of 1024 leaves little work between its two barriers.
// Bytes of a ring's row: where rows start anywhere, room for the granules that they share with their neighbours.
template <typename T>
__host__ __device__ constexpr uint32_t ring_slot(int dim, bool aligned) {
    const uint32_t bytes = static_cast<uint32_t>(dim) * sizeof(T);
    return aligned ? bytes : (bytes + 15) / 16 * 16 + 16;
}

template <typename T, Rows kRows, int kThreads, int KV>
__global__ void __launch_bounds__(kThreads) rms_bwd_ring_kernel(RmsBwdArgs a, int stages) {
    constexpr int VEC = VecOf<T>::kN;
    extern __shared__ __align__(128) unsigned char ring[];
    __shared__ float red[2][32];
    __shared__ uint64_t full[kRingStages];
    __shared__ int abort;
    const int t = threadIdx.x;
    const uint32_t row_bytes = static_cast<uint32_t>(a.dim) * sizeof(T), slot = ring_slot<T>(a.dim, kRows == kWhole);
    const int inputs = a.gh ? 3 : 2;
    const int64_t first = blockIdx.x, step = gridDim.x;
    // (kPhase: the rows of a CTA are a multiple of VEC apart, so its columns and weights stay the same)
    const int lead = kRows == kPhase ? static_cast<int>(first * a.dim % VEC) : 0;
    const int count = first < a.rows ? static_cast<int>((a.rows - 1 - first) / step) + 1 : 0;
    if (t == 0) {
        for (int s = 0; s < stages; ++s) tc::mbar_init(&full[s], 1);
        abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();
    auto start = [&](int i, int64_t r) {      // row r of h, gy or gh
        const void* p = i == 0 ? a.h : (i == 1 ? a.gy : a.gh);
        return reinterpret_cast<uintptr_t>(static_cast<const T*>(p) + r * (i == 0 ? a.ldh : (i == 1 ? a.ldgy : a.ldgh)));
    };
    auto load = [&](int j) {     // (thread 0) row j of this CTA
        const int s = j % stages;
        const int64_t r = first + j * step;
        const uint32_t dst = tc::smem_u32(ring) + s * 3 * slot, bar = tc::smem_u32(&full[s]);
        const uintptr_t src[3] = {start(0, r), start(1, r), start(2, r)};
        uint32_t bytes[3], all = 0;
#pragma unroll
        for (int i = 0; i < 3; ++i) {      // whole 16-byte granules
            bytes[i] = kRows == kWhole ? row_bytes : (static_cast<uint32_t>(src[i] & 15) + row_bytes + 15) & ~15u;
            if (i < inputs) all += bytes[i];
        }
        tc::mbar_expect_tx(&full[s], all);
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (i < inputs)
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                                 dst + i * slot),
                             "l"(src[i] & ~uintptr_t(15)), "r"(bytes[i]), "r"(bar)
                             : "memory");
    };
    if (t == 0)
        for (int j = 0; j < min(count, stages - 1); ++j) load(j);
    float acc[KV][VEC], w[KV][VEC];
#pragma unroll
    for (int k = 0; k < KV; ++k) {
        const int i = (k * kThreads + t) * VEC - lead;
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[k][e] = w[k][e] = 0.f;
        if (i < a.dim) load_w<T, kRows>(a.w, a.w_f32, i, a.dim, w[k]);
    }
    const float inv_dim = 1.f / static_cast<float>(a.dim);
    for (int j = 0; j < count; ++j) {
        const int s = j % stages;
        const int64_t r = first + j * step;
        const float rstd = a.rstd[r];
        const bool here = tc::mbar_wait(&full[s], (j / stages) & 1, &abort, a.wait_limit);
        const T* in[3];
#pragma unroll
        for (int i = 0; i < 3; ++i)
            in[i] = reinterpret_cast<const T*>(ring + (s * 3 + i) * slot + (kRows == kWhole ? 0 : start(i, r) & 15));
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < KV; ++k) {
            const int i = (k * kThreads + t) * VEC - lead;
            if (i < a.dim) {
                float h[VEC], g[VEC];
                Raw<T, kRows> v;
                v.load(in[0], i, a.dim);
                v.trim(i, a.dim);
                v.get(h);
                v.load(in[1], i, a.dim);
                v.trim(i, a.dim);
                v.get(g);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    acc[k][e] = fmaf(g[e], h[e] * rstd, acc[k][e]);
                    sum = fmaf(h[e], g[e] * w[k][e], sum);
                }
            }
        }
        if (!here) {
            abort = j + 1;
            atomicCAS(a.status, 0, 4);
        }
        sum = group_sum<kThreads>(sum, red[j & 1]);
        if (abort) break;                        // (seen by all after the barrier in group_sum)
        if (t == 0 && j + stages - 1 < count) load(j + stages - 1);
        const float c = sum * inv_dim * rstd * rstd * rstd;
#pragma unroll
        for (int k = 0; k < KV; ++k) {
            const int i = (k * kThreads + t) * VEC - lead;
            if (i < a.dim) {
                float h[VEC], g[VEC];
                Raw<T, kRows> v;
                v.load(in[0], i, a.dim);
                v.trim(i, a.dim);
                v.get(h);
                v.load(in[1], i, a.dim);
                v.trim(i, a.dim);
                v.get(g);
#pragma unroll
                for (int e = 0; e < VEC; ++e) g[e] = fmaf(rstd, g[e] * w[k][e], -c * h[e]);
                if (a.gh) {
                    v.load(in[2], i, a.dim);
                    v.trim(i, a.dim);
                    v.get(h);
#pragma unroll
                    for (int e = 0; e < VEC; ++e) g[e] += h[e];
                }
                v.set(g);
                v.store(static_cast<T*>(a.gx) + r * a.dim, i, a.dim);
            }
        }
    }
    if (abort && t == 0) {      // rows that are still on their way, from the one that did not come
        const unsigned long long deadline = tc::drain_deadline();
        for (int j = abort - 1; j < min(count, abort + stages - 2); ++j) tc::mbar_drain(&full[j % stages], (j / stages) & 1, deadline);
    }
    if (!a.partial) return;
    float* dst = a.partial + static_cast<int64_t>(blockIdx.x) * rms_partial_pitch(a.dim);
#pragma unroll
    for (int k = 0; k < KV; ++k) {
        const int i = (k * kThreads + t) * VEC - lead;
        if (kRows == kPhase) {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
                if (i + e >= 0 && i + e < a.dim) dst[i + e] = acc[k][e];
        } else if (i < a.dim) {
#pragma unroll
            for (int e = 0; e < VEC; e += 4)
                *reinterpret_cast<float4*>(dst + i + e) = make_float4(acc[k][e], acc[k][e + 1], acc[k][e + 2], acc[k][e + 3]);
        }
    }
}

// gw[c] = sum of the partial rows; 32 columns a CTA, 8 threads a column
template <typename T>
__global__ void __launch_bounds__(256) rms_gw_kernel(const float* __restrict__ partial, int rows, int dim,
                                                     void* __restrict__ gw, bool w_f32) {
    __shared__ float red[8][33];
    const int c = blockIdx.x * 32 + (threadIdx.x & 31), y = threadIdx.x >> 5;
    float s = 0.f;
    if (c < dim) {
#pragma unroll 8
        for (int r = y; r < rows; r += 8) s += partial[static_cast<int64_t>(r) * rms_partial_pitch(dim) + c];
    }
    red[y][threadIdx.x & 31] = s;
    __syncthreads();
    if (y == 0 && c < dim) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += red[j][threadIdx.x];
        if (w_f32) static_cast<float*>(gw)[c] = sum;
        else static_cast<T*>(gw)[c] = from_f<T>(sum);
    }
}

// Threads per row and vectors per thread for rows of `vecs` 16-byte vectors: the smallest group that holds them, a
// warp while a thread keeps at most 4.  kMore: sizes for widths of one vector more than a power of two (kPhase).
template <bool kLong, bool kMore, typename Fn>
cudaError_t by_width(int vecs, Fn&& fn) {
#define MMLTK_RMS_WIDTH(G, KV) \
    if (vecs <= G * KV) return fn(std::integral_constant<int, G>{}, std::integral_constant<int, KV>{})
    MMLTK_RMS_WIDTH(32, 1);
    MMLTK_RMS_WIDTH(32, 2);
    MMLTK_RMS_WIDTH(32, 4);
    MMLTK_RMS_WIDTH(128, 2);
    MMLTK_RMS_WIDTH(128, 4);
    if constexpr (kMore) MMLTK_RMS_WIDTH(192, 3);
    MMLTK_RMS_WIDTH(256, 4);
    if constexpr (kMore) MMLTK_RMS_WIDTH(384, 3);
    MMLTK_RMS_WIDTH(512, 4);
    if constexpr (kLong && kMore) MMLTK_RMS_WIDTH(768, 3);
    if constexpr (kLong) MMLTK_RMS_WIDTH(512, 8);      // fp32
#undef MMLTK_RMS_WIDTH
    return cudaErrorInvalidValue;
}

bool aligned(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace

cudaError_t launch_rms_fwd(Elt et, const RmsFwdArgs& a, cudaStream_t st) {
    if (a.rows <= 0) return cudaSuccess;
    if (a.dim <= 0 || a.dim > kRmsMaxDim) return cudaErrorInvalidValue;
    const bool quant = a.codes != nullptr;
    const int elems = quant ? static_cast<int>(mx_scale_tiles(a.fmt, a.dim)) * 4 * mx_block(a.fmt) : a.dim;
    const int64_t rows = quant ? (a.rows + 127) / 128 * 128 : a.rows;
    return MMLTK_DISPATCH_ELT(et, [&]() -> cudaError_t {
        using T = elt_t;
        constexpr int kN = VecOf<T>::kN;
        if (!aligned(a.w)) return cudaErrorInvalidValue;
        const bool whole = a.dim % kN == 0 && a.ldx % kN == 0 && aligned(a.x) &&
                           (!a.res || (a.ldr % kN == 0 && aligned(a.res)));
        const bool phase = (a.ldx - a.dim) % kN == 0 && aligned(a.x) && (!a.res || ((a.ldr - a.dim) % kN == 0 && aligned(a.res)));
        auto run = [&](auto mode) -> cudaError_t {
            constexpr Rows kRows = decltype(mode)::value;
            const int vecs = (elems + kN - 1) / kN + (kRows == kPhase);
            return by_width<sizeof(T) == 4, kRows == kPhase>(vecs, [&](auto gc, auto kc) -> cudaError_t {
                constexpr int G = decltype(gc)::value, KV = decltype(kc)::value;
                const int64_t per = G == 32 ? 8 : 1, blocks = (rows + per - 1) / per;
                if (blocks >= (int64_t(1) << 31)) return cudaErrorInvalidValue;
                const int threads = G == 32 ? 256 : G;
                const dim3 grid(static_cast<unsigned>(blocks));
                if (!quant) return launch_early(rms_fwd_kernel<T, kRows, G, KV, false>, grid, threads, st, 0, a);
                constexpr int kSmem = kRows == kPhase ? (G == 32 ? 256 : G) * KV * 16 : 0;
                constexpr auto kern = rms_fwd_kernel<T, kRows, G, KV, true>;
                static std::atomic<uint64_t> allowed{0};
                const cudaError_t e = kSmem > 48 * 1024 ? allow_smem(kern, allowed, kSmem) : cudaSuccess;
                return e != cudaSuccess ? e : launch_early(kern, grid, threads, st, kSmem, a);
            });
        };
        if (whole) return run(std::integral_constant<Rows, kWhole>{});
        if (phase && (elems + kN - 1) / kN < kRmsMaxDim / kN) return run(std::integral_constant<Rows, kPhase>{});
        return run(std::integral_constant<Rows, kAny>{});
    });
}

namespace {

template <typename T>
cudaError_t sum_gw(const RmsBwdArgs& a, int blocks, cudaStream_t st) {
    if (!a.partial) return cudaSuccess;
    rms_gw_kernel<T><<<(a.dim + 31) / 32, 256, 0, st>>>(a.partial, blocks, a.dim, a.gw, a.w_f32);
    return cudaGetLastError();
}

// Rows of more than two vectors a lane.  As many CTAs an SM as keep three stages (two from 24 KB a stage on): the
// barriers of one row are then under other rows' loads (16384 x 8192: 171 us with two CTAs of two stages, 189 with one
// of four; 65536 x 1024: 101 with eight CTAs, 123 with four).  Not for fp32 rows of over 9000 elements, whose two
// stages would not fit.
template <typename T, Rows kRows>
cudaError_t ring_bwd(const RmsBwdArgs& a, cudaStream_t st) {
    const int vecs = (a.dim + VecOf<T>::kN - 1) / VecOf<T>::kN + (kRows == kPhase);
    const int stage = 3 * static_cast<int>(ring_slot<T>(a.dim, kRows == kWhole));
    const int per_sm = vecs <= 128 ? 8 : (vecs <= 256 ? 6 : (3 * stage <= 72 * 1024 ? 3 : (2 * stage <= 108 * 1024 ? 2 : 1)));
    const int stages = std::min(kRingStages, kRingBytes / per_sm / stage);
    if (vecs <= 64 || vecs > 2048 || stages < 2) return cudaErrorNotSupported;
    // kPhase: rows of one offset in a CTA (one row, or rows a multiple of 8 apart)
    const int most = kRows == kPhase ? num_sms() * per_sm & ~7 : num_sms() * per_sm;
    const int blocks = static_cast<int>(std::min<int64_t>(a.rows, most));
    auto run = [&](auto tc, auto kc) -> cudaError_t {
        constexpr int kThreads = decltype(tc)::value, KV = decltype(kc)::value;
        static std::atomic<uint64_t> allowed{0};
        const cudaError_t e = allow_smem(rms_bwd_ring_kernel<T, kRows, kThreads, KV>, allowed, kRingBytes);
        if (e != cudaSuccess) return e;
        rms_bwd_ring_kernel<T, kRows, kThreads, KV><<<blocks, kThreads, stages * stage, st>>>(a, stages);
        const cudaError_t l = cudaGetLastError();
        return l != cudaSuccess ? l : sum_gw<T>(a, blocks, st);
    };
    using std::integral_constant;
    if (vecs <= 128) return run(integral_constant<int, 128>{}, integral_constant<int, 1>{});
    if (vecs <= 256) return run(integral_constant<int, 128>{}, integral_constant<int, 2>{});
    if (vecs <= 512) return run(integral_constant<int, 256>{}, integral_constant<int, 2>{});
    if (vecs <= 1024) return run(integral_constant<int, 256>{}, integral_constant<int, 4>{});
    if constexpr (kRows == kPhase)
        if (vecs <= 1152) return run(integral_constant<int, 384>{}, integral_constant<int, 3>{});
    return run(integral_constant<int, 512>{}, integral_constant<int, 4>{});
}

template <typename T, Rows kRows>
cudaError_t bwd(const RmsBwdArgs& a, bool phase, cudaStream_t st) {
    if (a.rows <= 0) return a.partial ? cudaMemsetAsync(a.gw, 0, a.dim * (a.w_f32 ? sizeof(float) : sizeof(T)), st) : cudaSuccess;
    cudaError_t e = phase ? ring_bwd<T, kPhase>(a, st) : cudaErrorNotSupported;
    if (e == cudaErrorNotSupported) e = ring_bwd<T, kRows>(a, st);
    if (e != cudaErrorNotSupported) return e;
    const int vecs = (a.dim + VecOf<T>::kN - 1) / VecOf<T>::kN;
    auto run = [&](auto kern, int rows_cta, int threads, int per_sm) -> cudaError_t {
        const int blocks = static_cast<int>(std::max<int64_t>(
            1, std::min<int64_t>((a.rows + rows_cta - 1) / rows_cta, static_cast<int64_t>(num_sms()) * per_sm)));
        kern<<<blocks, threads, 0, st>>>(a);
        const cudaError_t l = cudaGetLastError();
        return l != cudaSuccess ? l : sum_gw<T>(a, blocks, st);
    };
    if (vecs <= 32) return run(rms_bwd_kernel<T, kRows, 32, 1>, 8, 256, 3);
    if (vecs <= 64) return run(rms_bwd_kernel<T, kRows, 32, 2>, 8, 256, 3);
    if constexpr (sizeof(T) == 4) return run(rms_bwd_kernel<T, kRows, 1024, 4>, 1, 1024, 1);
    return cudaErrorInvalidValue;
}

}  // namespace

int rms_bwd_partials(int64_t rows) {
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(rows, num_sms() * 8)));
}

cudaError_t launch_rms_bwd(Elt et, const RmsBwdArgs& a, cudaStream_t st) {
    if (a.dim <= 0 || a.dim > kRmsMaxDim || !aligned(a.w)) return cudaErrorInvalidValue;
    return MMLTK_DISPATCH_ELT(et, [&]() -> cudaError_t {
        using T = elt_t;
        constexpr int kN = VecOf<T>::kN;
        const bool whole = a.dim % kN == 0 && aligned(a.h) && a.ldh % kN == 0 && a.ldgy % kN == 0 && aligned(a.gy) &&
                           (!a.gh || (a.ldgh % kN == 0 && aligned(a.gh)));
        const bool phase = (a.ldh - a.dim) % kN == 0 && aligned(a.h) && (a.ldgy - a.dim) % kN == 0 && aligned(a.gy) &&
                           (!a.gh || ((a.ldgh - a.dim) % kN == 0 && aligned(a.gh)));
        return whole ? bwd<T, kWhole>(a, false, st) : bwd<T, kAny>(a, phase, st);
    });
}

}  // namespace mmltk
