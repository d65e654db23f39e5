// Product of two microscaled matrices on the block-scaled tensor cores:
//
//   y[m, n] = act(g_x g_w sum_k (x[m, k] s_x[m, k / B]) (w[n, k] s_w[n, k / B]) + bias[n])
//
// tcgen05.mma with .block_scale multiplies the 4- or 8-bit elements and their scales inside the
// tensor core and accumulates in fp32 in tensor memory; neither operand is ever expanded.  One
// kernel for the three formats: a row of an operand tile is 128 bytes of codes (256 4-bit or 128
// 8-bit elements) in the 128-byte swizzle, one MMA takes 32 bytes of it, and only the instruction's
// kind and the place of its scales differ:
//   nvfp4  kind::mxf4nvf4, 4 scales per row and MMA: one 128 x 4 scale tile per MMA
//   mxfp4  kind::mxf4,     2 scales: half a tile, chosen by the descriptor's scale id 0 / 2
//   mxfp8  kind::mxf8f6f4, 1 scale:  a quarter, id 0 .. 3
//
// Persistent, ten warps: warp 0 loads (TMA: codes as 128-byte swizzled boxes, scale tiles as 512-byte
// rows), warp 1 copies each stage's scales to tensor memory (tcgen05.cp, ordered before the MMAs of the
// same thread) and issues the MMAs, warps 2-9 are the epilogue.  Two accumulators let it run under the
// next tile's products.  With 256 columns two accumulators and the scales do not fit the 512 columns of
// tensor memory: the second starts at column 208, and the epilogue drains the 48 shared columns first.
//
// The quantised output (mxfp8) needs no second pass: a thread holds 32 consecutive columns of a row,
// which are one scale block.
//
// Every wait is bounded: on a time-out the kernel records which role gave up in a status word and
// leaves, after releasing its tensor memory.
#include <cudaTypedefs.h>

#include <cstdio>

#include "microscale.cuh"
#include "tcgen05.cuh"

namespace mmltk {

namespace {

using namespace mx;
using namespace tc;

constexpr int kThreads = 320;
constexpr int kEpiWarps = 8;
constexpr int kRowBytes = 128;                     // bytes of codes per row and stage
constexpr int kATile = 128 * kRowBytes;
constexpr int kStageTile = 32 * 64;                // staging of one 32-row chunk of the output
constexpr int kMaxStages = 6;
constexpr int kSmemMax = 227 * 1024;

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

template <MxFormat F>
__device__ __forceinline__ void mma_block(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa,
                                          uint32_t sfb, uint32_t accumulate) {
    if constexpr (F == MxFormat::kNvFp4) {
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate));
    } else if constexpr (F == MxFormat::kMxFp4) {
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate));
    } else {
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate));
    }
}

// One 32 x 16 byte scale tile from shared memory to 4 columns of tensor memory, in all four lane quarters.
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint32_t smem) {
    uint64_t d = static_cast<uint64_t>((smem >> 4) & 0x3fff);
    d |= static_cast<uint64_t>(128 >> 4) << 32;       // 8-row groups 128 bytes apart; one 16-byte column
    d |= 1ull << 46;
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
}

__device__ __forceinline__ void tma_load_3d(const CUtensorMap* map, uint64_t* bar, void* dst, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}

template <MxFormat F, int BN_>
struct Cfg {
    static constexpr int BN = BN_;
    static constexpr int kAtoms = Kind<F>::kAtoms;
    static constexpr int kBTile = BN * kRowBytes;
    static constexpr int kSfA = kAtoms * 512;
    static constexpr int kSfB = (BN / 128) * kAtoms * 512;
    static constexpr int kStageBytes = kATile + kBTile + kSfA + kSfB;
    static constexpr int kFixed = kEpiWarps * kStageTile + kEpiWarps * (BN / 2) * 4 + 1024 + 256;
    static constexpr int kStages =
        (kSmemMax - kFixed) / kStageBytes < kMaxStages ? (kSmemMax - kFixed) / kStageBytes : kMaxStages;
    static constexpr size_t kSmemBytes = static_cast<size_t>(kStages) * kStageBytes + kFixed;
    // tensor memory columns: accumulators at 0 and kAcc1, scales from kSfCol
    static constexpr int kSfCols = kAtoms * 4 * (1 + BN / 128);
    static constexpr int kTmemCols = BN == 256 ? 512 : 512;
    static constexpr int kSfCol = 512 - 48;
    static constexpr int kAcc1 = BN == 256 ? kSfCol - 256 : 128;
    static constexpr bool kOverlap = BN == 256;
    static_assert(kSfCols <= 48);
};

struct __align__(8) Ctl {
    uint64_t full[kMaxStages];
    uint64_t empty[kMaxStages];
    uint64_t acc_full[2];
    uint64_t acc_empty[2];
    uint64_t shared_empty[2];     // the columns that both accumulators use have been read
    uint32_t tmem_base;
    int abort;
};

struct Sched {
    int m_tiles, n_tiles, ktiles, units;
    // groups of 8 row tiles, column-major inside a group: the tiles in flight share operand rows in L2
    __device__ void tile(int u, int& mt, int& nt) const {
        const int per = 8 * n_tiles, g = u / per, rest = u % per;
        const int height = min(8, m_tiles - 8 * g);
        mt = 8 * g + rest % height;
        nt = rest / height;
    }
};

// Output of one warp's 32 x 32 chunk (lane = row).
template <typename O>
struct Out {
    static constexpr int kCols = 64 / sizeof(O);       // columns of a 64-byte staging row: 32 or 16
};

template <typename O>
__device__ __forceinline__ void store_chunk(const MxGemmArgs& g, unsigned char* buf, const CUtensorMap* map, bool tma,
                                            int lane, const float* x, int col, int row0) {
    constexpr int kCols = Out<O>::kCols;
#pragma unroll
    for (int part = 0; part < 32 / kCols; ++part) {
        const int c0 = col + part * kCols;
        if (c0 >= g.n) break;
        if (tma && lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
        __syncwarp();
        unsigned char* rowp = buf + lane * 64;
        const int sw = (lane >> 1) & 3;     // 64-byte swizzle
#pragma unroll
        for (int c = 0; c < 4; ++c)
            *reinterpret_cast<uint4*>(rowp + ((c ^ sw) << 4)) = pack16(x + part * kCols + c * (16 / sizeof(O)), O());
        if (tma) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map),
                             "r"(smem_u32(buf)), "r"(c0), "r"(row0)
                             : "memory");
                asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            }
        } else {
            // rows that are no multiple of 16 bytes: 64-byte row segments, a lane per element
            __syncwarp();
            for (int r = 0; r < 32 && row0 + r < g.m; ++r)
                for (int e = lane; e < kCols && c0 + e < g.n; e += 32) {
                    const int byte = e * static_cast<int>(sizeof(O));
                    const O* p = reinterpret_cast<const O*>(buf + r * 64 + (((byte >> 4) ^ ((r >> 1) & 3)) << 4) + (byte & 15));
                    static_cast<O*>(g.y)[static_cast<int64_t>(row0 + r) * g.n + c0 + e] = *p;
                }
            __syncwarp();
        }
    }
}

// mxfp8 output: the 32 columns are one scale block.  Returns the scale byte.
__device__ __forceinline__ uint32_t store_chunk_q(const MxGemmArgs& g, unsigned char* buf, const CUtensorMap* map,
                                                  int lane, float* x, int col, int row0) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        if (col + i >= g.n) x[i] = 0.f;
        m = max(m, abs_bits(x[i]));
    }
    const BlockScale sc = pow2_scale<8>(__uint_as_float(m));
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
    uint4* rowp = reinterpret_cast<uint4*>(buf + lane * 32);
#pragma unroll
    for (int c = 0; c < 2; ++c)
        rowp[c] = make_uint4(cvt_e4m3x4(x + 16 * c, sc.inv), cvt_e4m3x4(x + 16 * c + 4, sc.inv),
                             cvt_e4m3x4(x + 16 * c + 8, sc.inv), cvt_e4m3x4(x + 16 * c + 12, sc.inv));
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) {
        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map),
                     "r"(smem_u32(buf)), "r"(col), "r"(row0)
                     : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
    return sc.byte;
}

template <MxFormat F, int BN_, typename O, bool kQuantOut>
__global__ void __launch_bounds__(kThreads, 1)
    mx_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                   const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB,
                   const __grid_constant__ CUtensorMap tmY, MxGemmArgs g, Sched sch, bool tma_store) {
    using C = Cfg<F, BN_>;
    using K = Kind<F>;
    constexpr int BN = C::BN, kStages = C::kStages, kAtoms = C::kAtoms;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* tilesA = smem;
    unsigned char* tilesB = tilesA + kStages * kATile;
    unsigned char* sfA = tilesB + kStages * C::kBTile;
    unsigned char* sfB = sfA + kStages * C::kSfA;
    unsigned char* staging = sfB + kStages * C::kSfB;
    float* bias_s = reinterpret_cast<float*>(staging + kEpiWarps * kStageTile);
    Ctl* ctl = reinterpret_cast<Ctl*>(bias_s + kEpiWarps * (BN / 2));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&ctl->full[s], 1);
            mbar_init(&ctl->empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&ctl->acc_full[b], 1);
            mbar_init(&ctl->acc_empty[b], kEpiWarps);
            mbar_init(&ctl->shared_empty[b], kEpiWarps / 2);
        }
        ctl->abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl->tmem_base)),
                     "r"(C::kTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = ctl->tmem_base;

    if (warp == 0) {
        if (lane == 0) {
            int it = 0;
            for (int u = blockIdx.x; u < sch.units; u += gridDim.x) {
                int mt, nt;
                sch.tile(u, mt, nt);
                for (int kt = 0; kt < sch.ktiles; ++kt, ++it) {
                    const int s = it % kStages;
                    if (!mbar_wait(&ctl->empty[s], ((it / kStages) & 1) ^ 1, &ctl->abort)) {
                        ctl->abort = 1;
                        atomicCAS(g.status, 0, 1);
                        goto producer_done;
                    }
                    // boxes past an extent are zero-filled and count in full
                    mbar_expect_tx(&ctl->full[s], C::kStageBytes);
                    tma_load_2d(&tmA, &ctl->full[s], tilesA + s * kATile, kt * kRowBytes, mt * 128);
                    tma_load_2d(&tmB, &ctl->full[s], tilesB + s * C::kBTile, kt * kRowBytes, nt * BN);
                    tma_load_3d(&tmSA, &ctl->full[s], sfA + s * C::kSfA, 0, kt * kAtoms, mt);
                    tma_load_3d(&tmSB, &ctl->full[s], sfB + s * C::kSfB, 0, kt * kAtoms, nt * (BN / 128));
                }
            }
        producer_done:;
        }
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = K::kDesc | (static_cast<uint32_t>(BN >> 3) << 17) | (128u >> 4 << 24);
            const uint32_t tsa = tmem + C::kSfCol, tsb = tsa + 4 * kAtoms;
            int it = 0, local = 0;
            for (int u = blockIdx.x; u < sch.units; u += gridDim.x, ++local) {
                const int buf = local & 1;
                bool ok = mbar_wait(&ctl->acc_empty[buf], ((local >> 1) & 1) ^ 1, &ctl->abort);
                if (C::kOverlap && local > 0)
                    ok = ok && mbar_wait(&ctl->shared_empty[buf ^ 1], ((local - 1) >> 1) & 1, &ctl->abort);
                if (!ok) {
                    ctl->abort = 1;
                    atomicCAS(g.status, 0, 2);
                    break;
                }
                tc_fence_after();
                const uint32_t acc = tmem + buf * C::kAcc1;
                for (int kt = 0; kt < sch.ktiles; ++kt, ++it) {
                    const int s = it % kStages;
                    if (!mbar_wait(&ctl->full[s], (it / kStages) & 1, &ctl->abort)) {
                        ctl->abort = 1;
                        atomicCAS(g.status, 0, 2);
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t a = smem_u32(tilesA + s * kATile), b = smem_u32(tilesB + s * C::kBTile);
                    const uint32_t pa = smem_u32(sfA + s * C::kSfA), pb = smem_u32(sfB + s * C::kSfB);
                    // scale tile j: A at columns tsa + 4 j; B's row tiles side by side for each j
#pragma unroll
                    for (int j = 0; j < kAtoms; ++j) {
                        copy_scales(tsa + 4 * j, pa + j * 512);
#pragma unroll
                        for (int r = 0; r < BN / 128; ++r)
                            copy_scales(tsb + (BN / 128) * 4 * j + 4 * r, pb + (r * kAtoms + j) * 512);
                    }
                    // MMAs that only see padding are left out (their scales may be another row tile's)
                    const int mmas = min(4, (g.k - kt * K::kElems + K::kElems / 4 - 1) / (K::kElems / 4));
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        if (kk < mmas) {
                            const int j = kk * kAtoms / 4;
                            const uint32_t id = F == MxFormat::kNvFp4 ? 0u : (F == MxFormat::kMxFp4 ? (kk & 1) * 2u : kk);
                            mma_block<F>(acc, operand_desc<false>(a, kk), operand_desc<false>(b, kk),
                                         idesc | (id << 4) | (id << 29), tsa + 4 * j, tsb + (BN / 128) * 4 * j,
                                         (kt | kk) ? 1u : 0u);
                        }
                    }
                    tc_commit(&ctl->empty[s]);
                }
                if (!ok) break;
                tc_commit(&ctl->acc_full[buf]);
            }
        }
    } else {
        const int q = warp & 3, half = (warp - 2) >> 2;
        constexpr int kHalf = BN / 2, kChunks = kHalf / 32;
        unsigned char* buf_s = staging + (warp - 2) * kStageTile;
        float* bias_w = bias_s + (warp - 2) * kHalf;
        const float alpha = (g.x_g ? *g.x_g : 1.f) * (g.w_g ? *g.w_g : 1.f);
        const int ykt = kQuantOut ? static_cast<int>(mx_scale_tiles(MxFormat::kMxFp8, g.n)) : 0;
        int local = 0;
        for (int u = blockIdx.x; u < sch.units; u += gridDim.x, ++local) {
            int mt, nt;
            sch.tile(u, mt, nt);
            const int row0 = mt * 128 + 32 * q, col0 = nt * BN + half * kHalf;
            // this warp's columns of the bias, as fp32
            __syncwarp();
            for (int i = lane; i < kHalf; i += 32) {
                float b = 0.f;
                if (g.bias && col0 + i < g.n)
                    b = g.bias_elt == Elt::kF32 ? static_cast<const float*>(g.bias)[col0 + i]
                        : g.bias_elt == Elt::kBF16 ? to_f(static_cast<const __nv_bfloat16*>(g.bias)[col0 + i])
                                                   : to_f(static_cast<const __half*>(g.bias)[col0 + i]);
                bias_w[i] = b;
            }
            __syncwarp();
            const int buf = local & 1;
            if (!mbar_wait(&ctl->acc_full[buf], (local >> 1) & 1, &ctl->abort)) {
                if (lane == 0) atomicCAS(g.status, 0, 3);
                ctl->abort = 1;
                break;
            }
            tc_fence_after();
            const uint32_t acc = tmem + buf * C::kAcc1 + (static_cast<uint32_t>(32 * q) << 16) + half * kHalf;
            // the two chunks with columns that both accumulators use come first: the last two of the
            // first accumulator's right half, the first two of the second's left half
            const bool shares = C::kOverlap && half == (buf ^ 1);
            const int first = (shares && buf == 0) ? kChunks - 2 : 0;
            uint32_t bytes = 0;
#pragma unroll 1
            for (int i = 0; i < kChunks; ++i) {
                const int c = (first + i) & (kChunks - 1);
                const int col = col0 + 32 * c;
                const bool live = col < g.n && row0 < g.m;
                float v[32];
                tmem_ld32(acc + 32 * c, v);
                if (shares && i == 1) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ctl->shared_empty[buf]);
                }
                if (i == kChunks - 1) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ctl->acc_empty[buf]);
                }
                uint32_t byte = 0;
                if (live) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float4 b = reinterpret_cast<const float4*>(bias_w + 32 * c)[j];
                        v[4 * j] = fmaf(v[4 * j], alpha, b.x);
                        v[4 * j + 1] = fmaf(v[4 * j + 1], alpha, b.y);
                        v[4 * j + 2] = fmaf(v[4 * j + 2], alpha, b.z);
                        v[4 * j + 3] = fmaf(v[4 * j + 3], alpha, b.w);
                    }
                    if (g.act == 1) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = gelu_fwd(v[j]);
                    } else if (g.act == 2) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) v[j] = fmaxf(v[j], 0.f);
                    }
                    if constexpr (kQuantOut) {
                        byte = store_chunk_q(g, buf_s, &tmY, lane, v, col, row0);
                        if (row0 + lane >= g.m) byte = 0;
                    } else {
                        store_chunk<O>(g, buf_s, &tmY, tma_store, lane, v, col, row0);
                    }
                }
                if constexpr (kQuantOut) bytes |= byte << (8 * (c & 3));
            }
            if constexpr (kQuantOut) {
                // scale bytes of this row's blocks: four (two) neighbours, one store; zero past m and n
                if (nt * BN / 128 + half * kHalf / 128 < ykt) {
                    uint8_t* p = static_cast<uint8_t*>(g.scales) + scale_offset(row0 + lane, col0 / 32, ykt);
                    if constexpr (kChunks == 4) *reinterpret_cast<uint32_t*>(p) = bytes;
                    else *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(bytes);
                }
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::kTmemCols));
    }
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
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
bool codes_map(CUtensorMap* map, const void* p, int64_t row_bytes, int64_t rows, int64_t pitch, int box_rows) {
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
bool scales_map(CUtensorMap* map, const void* p, int64_t rows, int kt, int atoms, int row_tiles) {
    auto fn = encode_fn();
    if (!fn) return false;
    cuuint64_t dims[3] = {256, static_cast<cuuint64_t>(kt), static_cast<cuuint64_t>((rows + 127) / 128)};
    cuuint64_t strides[2] = {512, static_cast<cuuint64_t>(kt) * 512};
    cuuint32_t box[3] = {256, static_cast<cuuint32_t>(atoms), static_cast<cuuint32_t>(row_tiles)}, es[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(p), dims, strides, box, es,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Output: 32-row boxes of 64 bytes (64-byte swizzle) or, quantised, of 32 codes; stores past the extents are clipped.
bool out_map(CUtensorMap* map, void* p, Elt e, bool quant, int64_t cols, int64_t rows, int64_t pitch) {
    auto fn = encode_fn();
    if (!fn) return false;
    const CUtensorMapDataType dt = quant ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : e == Elt::kF32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : e == Elt::kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                    : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch)};
    cuuint32_t box[2] = {(!quant && e == Elt::kF32) ? 16u : 32u, 32u}, es[2] = {1, 1};
    return fn(map, dt, 2, p, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
              quant ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <MxFormat F, int BN, typename O, bool kQ>
cudaError_t launch(const MxGemmArgs& g, cudaStream_t st) {
    using C = Cfg<F, BN>;
    CUtensorMap ta, tb, sa, sb, ty{};
    const int64_t row_bytes = (static_cast<int64_t>(g.k) * mx_bits(F) + 7) / 8;
    const int kt = static_cast<int>(mx_scale_tiles(F, g.k));
    const bool tma_store = kQ || (g.y_pitch % 16 == 0 && reinterpret_cast<uintptr_t>(g.y) % 16 == 0);
    bool ok = codes_map(&ta, g.x_codes, row_bytes, g.m, g.x_pitch, 128) &&
              codes_map(&tb, g.w_codes, row_bytes, g.n, g.w_pitch, BN) &&
              scales_map(&sa, g.x_scales, g.m, kt, C::kAtoms, 1) &&
              scales_map(&sb, g.w_scales, g.n, kt, C::kAtoms, BN / 128);
    if (kQ) ok = ok && out_map(&ty, g.codes, g.out, true, g.y_pitch, g.m, g.y_pitch);
    else if (tma_store) ok = ok && out_map(&ty, g.y, g.out, false, g.n, g.m, g.y_pitch);
    if (!ok) return cudaErrorInvalidValue;
    Sched sch;
    sch.m_tiles = (g.m + 127) / 128;
    sch.n_tiles = (g.n + BN - 1) / BN;
    sch.ktiles = (g.k + Kind<F>::kElems - 1) / Kind<F>::kElems;
    sch.units = sch.m_tiles * sch.n_tiles;
    auto kern = mx_gemm_kernel<F, BN, O, kQ>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(C::kSmemBytes));
    if (e != cudaSuccess) return e;
    kern<<<std::min(sch.units, num_sms()), kThreads, C::kSmemBytes, st>>>(ta, tb, sa, sb, ty, g, sch, tma_store);
    return cudaGetLastError();
}

template <MxFormat F, int BN>
cudaError_t by_output(const MxGemmArgs& g, cudaStream_t st) {
    if (g.codes) return launch<F, BN, float, true>(g, st);
    if (g.out == Elt::kBF16) return launch<F, BN, __nv_bfloat16, false>(g, st);
    if (g.out == Elt::kF16) return launch<F, BN, __half, false>(g, st);
    return launch<F, BN, float, false>(g, st);
}

template <MxFormat F>
cudaError_t by_tile(const MxGemmArgs& g, cudaStream_t st) {
    // 256-column tiles move a third fewer operand bytes per product; 128 where they would leave SMs idle
    const int64_t wide = static_cast<int64_t>((g.m + 127) / 128) * ((g.n + 255) / 256);
    if (g.n > 128 && wide >= num_sms()) return by_output<F, 256>(g, st);
    return by_output<F, 128>(g, st);
}

}  // namespace

cudaError_t launch_mx_gemm(const MxGemmArgs& g, cudaStream_t st) {
    if (g.m <= 0 || g.n <= 0 || g.k <= 0) return cudaErrorInvalidValue;
    // the tensor maps are encoded through the driver API, which needs a current context
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaSetDevice(dev);
    if (e != cudaSuccess) return e;
    if (g.fmt == MxFormat::kMxFp4) return by_tile<MxFormat::kMxFp4>(g, st);
    if (g.fmt == MxFormat::kNvFp4) return by_tile<MxFormat::kNvFp4>(g, st);
    return by_tile<MxFormat::kMxFp8>(g, st);
}

}  // namespace mmltk
