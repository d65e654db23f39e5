// Product of few tokens (at most 32) with a microscaled weight, in one launch:
//
//   y[t, n] = act(g_x g_w sum_k x_q[t, k] w[n, k] + bias[n])
//
// Bound by the weight's bytes (4-bit: n k / 2 + scales, 1.4 us for 4096 x 4096) and, below some
// microseconds, by latency.  So the roles are swapped -- 128 weight rows are the MMA's rows, the
// tokens its columns -- and the reduction is cut into up to 8 slices, the CTAs of a cluster, so
// that small weights still have CTAs on every SM and every CTA's stages are in flight at once.
// While its weight stages travel, each CTA quantises its slice of x into the swizzled operand
// layout itself (a separate pass would cost a launch; the slices are quantised once per row tile,
// by CTAs that would be waiting).  Each CTA's partial sums (fp32, tensor memory) go to its shared
// memory; after a cluster barrier the CTAs add the slices in their order, each a part of the
// outputs, reading the others' shared memory.  No atomics, no workspace: the same bits every run.
//
// Measured, one token, graph replays: nvfp4 4096 x 4096 5.8 to 6.0 us (17 as a quantisation and 128-row tiles); mxfp8
// 8192 x 8192 17.0 us (4.1 TB/s) with weights in turn, 14.8 with one, which stays in L2.  What is left above the weight's
// 1.4 and 10.6 us is set-up, one load latency (the first load waits for the kernel in front), the partial sums' way
// through shared memory and two cluster barriers.
//
// Waits are bounded; on a time-out the kernel sets the status word and leaves.
#include "mx_mma.cuh"

namespace mmltk {

namespace {

using namespace mx;

constexpr int kFewThreads = 256;
constexpr int kFewSplits = 8;          // portable cluster size
constexpr int kFewStages = 5;
constexpr int kWTile = 128 * kRowBytes;
constexpr int kFewSmemMax = 112 * 1024;      // two CTAs an SM

struct FewPlan {
    int splits, kt_per, ktiles, stages;
    uint32_t b_off, sfb_off, ctl_off, smem;      // shared memory: weight stages (codes, scales), x's codes, x's scales
};

struct __align__(8) FewCtl {
    uint64_t full[kFewStages], empty[kFewStages], done, drained;
    uint32_t tmem_base;
    int abort;
};

__device__ __forceinline__ float ld_cluster(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
    return v;
}

// kTok: tokens padded to the MMA's N (8, 16 or 32).  T: x's element type, or uint8_t for quantised x.
template <MxFormat F, int kTok, typename T>
__global__ void __launch_bounds__(kFewThreads, 2)
    mx_few_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmSW, MxFewArgs a,
                  FewPlan pl, int align) {
    using K = Kind<F>;
    using Tr = Traits<F>;
    constexpr int kAtoms = K::kAtoms, kStage = kWTile + kAtoms * 512, kBTile = kTok * kRowBytes;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* sfw = smem + pl.stages * kWTile;
    unsigned char* xs = smem + pl.b_off;
    unsigned char* sfx = smem + pl.sfb_off;
    FewCtl* ctl = reinterpret_cast<FewCtl*>(smem + pl.ctl_off);
    const MxGemmArgs& g = a.g;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rank = blockIdx.x % pl.splits, nt = blockIdx.x / pl.splits;
    const int kt0 = rank * pl.kt_per, kts = max(0, min(pl.kt_per, pl.ktiles - kt0));

    if (threadIdx.x == 0) {
        for (int s = 0; s < kFewStages; ++s) {
            mbar_init(&ctl->full[s], 1);
            mbar_init(&ctl->empty[s], 1);
        }
        mbar_init(&ctl->done, 1);
        mbar_init(&ctl->drained, 1);
        ctl->abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl->tmem_base)),
                     "r"(128));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    wait_previous();
    allow_next();
    const uint32_t tmem = ctl->tmem_base;
    const uint32_t elected = elect_lane();

    auto load_stage = [&](int i) {      // warp 0: weight stage i of this slice
        const int s = i % pl.stages;
        if (elected) mbar_expect_tx(&ctl->full[s], kStage);
        const uint32_t bar = smem_u32(&ctl->full[s]);
        load_2d<false>(elected, &tmW, bar, smem_u32(smem + s * kWTile), (kt0 + i) * kRowBytes, nt * 128);
        load_3d<false>(elected, &tmSW, bar, smem_u32(sfw + s * kAtoms * 512), 0, (kt0 + i) * kAtoms, nt);
    };
    if (warp == 0)
        for (int i = 0; i < min(kts, pl.stages); ++i) load_stage(i);

    // x's slice: codes as kTok rows of 128 bytes a stage (16-byte pieces swizzled by row), scales as scale tiles
    if constexpr (std::is_same_v<T, uint8_t>) {
        const uint8_t* codes = static_cast<const uint8_t*>(g.x_codes);
        for (int i = threadIdx.x; i < kts * g.m * 8; i += kFewThreads) {
            const int piece = i & 7, t = (i >> 3) % g.m, st = (i >> 3) / g.m;
            const int64_t byte = static_cast<int64_t>(kt0 + st) * kRowBytes + piece * 16;
            uint4 w = make_uint4(0, 0, 0, 0);
            if (byte < g.x_pitch) w = *reinterpret_cast<const uint4*>(codes + t * g.x_pitch + byte);
            *reinterpret_cast<uint4*>(xs + st * kBTile + t * kRowBytes + ((piece ^ (t & 7)) << 4)) = w;
        }
        const int64_t tiles = mx_scale_tiles(F, g.k);
        for (int i = threadIdx.x; i < kts * kAtoms * 32; i += kFewThreads) {
            const int64_t tile = static_cast<int64_t>(kt0) * kAtoms + i / 32;
            uint4 w = make_uint4(0, 0, 0, 0);
            if (tile < tiles) w = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(g.x_scales) + tile * 512)[i % 32];
            reinterpret_cast<uint4*>(sfx)[i] = w;
        }
    } else {
        constexpr int kParts = K::kElems / 16;      // 16-element parts of a row and stage
        const float gx = (!Tr::kPow2 && g.x_g) ? *g.x_g : 1.f;
        // a thread keeps its part of the row and walks (stage, token); the loads of kAhead steps are in flight together
        constexpr int kAhead = 2, kStep = kFewThreads / kParts;
        const int part = threadIdx.x % kParts, total = kts * g.m;
        int st = 0, t = threadIdx.x / kParts;
        const int first = t;
        while (t >= g.m && st < kts) {
            t -= g.m;
            ++st;
        }
        for (int i0 = 0; i0 < total; i0 += kAhead * kStep) {
            Raw16<T> raw[kAhead];
            int ts[kAhead], sts[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                ts[u] = t;
                sts[u] = st;
                if (i0 + u * kStep + first < total)
                    raw[u].load(static_cast<const T*>(a.x) + t * a.ldx, (kt0 + st) * K::kElems + part * 16, g.k, align);
                else
                    raw[u].zero();
                t += kStep;
                while (t >= g.m && st < kts) {
                    t -= g.m;
                    ++st;
                }
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const bool live = i0 + u * kStep + first < total;
                uint32_t m = raw[u].amax_bits();
                if constexpr (Tr::kBlock == 32) m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
                if (!live) continue;
                float v[16];
                raw[u].get(v);
                const BlockScale sc = block_scale<F>(__uint_as_float(m), gx);
                unsigned char* row = xs + sts[u] * kBTile + ts[u] * kRowBytes;
                if constexpr (Tr::kBits == 4) {
                    *reinterpret_cast<uint2*>(row + (((part >> 1) ^ (ts[u] & 7)) << 4) + (part & 1) * 8) =
                        make_uint2(cvt_e2m1x8(v, sc.inv), cvt_e2m1x8(v + 8, sc.inv));
                } else {
                    *reinterpret_cast<uint4*>(row + ((part ^ (ts[u] & 7)) << 4)) =
                        make_uint4(cvt_e4m3x4(v, sc.inv), cvt_e4m3x4(v + 4, sc.inv), cvt_e4m3x4(v + 8, sc.inv),
                                   cvt_e4m3x4(v + 12, sc.inv));
                }
                const int b = part * 16 / Tr::kBlock;
                if (Tr::kBlock == 16 || (part & 1) == 0)
                    sfx[(sts[u] * kAtoms + (b >> 2)) * 512 + (ts[u] & 31) * 16 + (ts[u] >> 5) * 4 + (b & 3)] =
                        static_cast<uint8_t>(sc.byte);
            }
        }
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();

    if (warp == 0) {
        // the remaining weight stages as the first ones are used up (one warp: MMAs of stage i, then the reload)
        constexpr uint32_t idesc = K::kDesc | (static_cast<uint32_t>(kTok >> 3) << 17) | (128u >> 4 << 24);
        bool ok = true;
        int loaded = 0;
        for (int i = 0; i < kts; ++i) {
            const int s = i % pl.stages;
            ok = __all_sync(0xffffffffu, mbar_wait(&ctl->full[s], (i / pl.stages) & 1, &ctl->abort, g.wait_limit));
            loaded = i + pl.stages;
            if (!ok) break;
            tc_fence_after();
            const uint32_t wa = operand_lo(smem_u32(smem + s * kWTile)), xb = operand_lo(smem_u32(xs + i * kBTile));
            const uint32_t pw = smem_u32(sfw + s * kAtoms * 512) >> 4, px = smem_u32(sfx + i * kAtoms * 512) >> 4;
            const uint32_t tsw = tmem + 64 + (i & 1) * 32, tsx = tsw + 4 * kAtoms;
#pragma unroll
            for (int j = 0; j < kAtoms; ++j) {
                copy_scales<false>(elected, tsw + 4 * j, pw + j * 32);
                copy_scales<false>(elected, tsx + 4 * j, px + j * 32);
            }
            const int left = g.k - (kt0 + i) * K::kElems;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
                if (kk * (K::kElems / 4) < left) {
                    const int j = kk * kAtoms / 4;
                    const uint32_t id = F == MxFormat::kNvFp4 ? 0u : (F == MxFormat::kMxFp4 ? (kk & 1) * 2u : kk);
                    mma_block<F, false>(elected, tmem, wa + 2 * kk, xb + 2 * kk, idesc | (id << 4) | (id << 29),
                                        tsw + 4 * j, tsx + 4 * j, (i | kk) ? 1u : 0u);
                }
            commit<false>(elected, smem_u32(&ctl->empty[s]));
            if (i + pl.stages < kts) {
                ok = __all_sync(0xffffffffu, mbar_wait(&ctl->empty[s], (i / pl.stages) & 1, &ctl->abort));
                if (!ok) break;
                load_stage(i + pl.stages);
            }
        }
        if (ok && kts > 0) commit<false>(elected, smem_u32(&ctl->done));
        if (!ok) {
            if (elected) {
                ctl->abort = 1;
                atomicCAS(g.status, 0, 2);
            }
            // the loads and products that are under way end before anything else happens to their memory
            commit<false>(elected, smem_u32(&ctl->drained));
            const unsigned long long deadline = drain_deadline();
            for (int i = max(0, loaded - pl.stages); i < min(kts, loaded); ++i)
                mbar_drain(&ctl->full[i % pl.stages], (i / pl.stages) & 1, deadline);
            mbar_drain(&ctl->drained, 0, deadline);
            __syncwarp();
        }
    }
    // partial sums to shared memory (over the weight stages, which nothing reads any more): part[t][row]
    float* part = reinterpret_cast<float*>(smem);
    bool good = true;
    if (kts > 0) {
        good = mbar_wait(&ctl->done, 0, &ctl->abort);
        tc_fence_after();
    }
    good = __syncthreads_and(good);
    if (!good && threadIdx.x == 0) atomicCAS(g.status, 0, 3);
    if (warp < 4) {
#pragma unroll
        for (int c = 0; c < kTok; c += 8) {
            uint32_t r[8] = {};
            if (kts > 0) {      // (the same for the whole CTA)
                asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                             : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                             : "r"(tmem + c + (static_cast<uint32_t>(32 * warp) << 16)));
                asm volatile("tcgen05.wait::ld.sync.aligned;"
                             : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])
                             :
                             : "memory");
            }
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < g.m) part[(c + e) * 128 + 32 * warp + lane] = __uint_as_float(r[e]);
        }
    }
    tc_fence_before();
    __syncthreads();
    // tensor memory is given back before this CTA waits for its cluster: a CTA that held some could wait for one that
    // cannot get any, behind a kernel of another stream that in turn waits for this CTA's
    if (warp == 0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(128));
    }
    cluster_sync_all();

    // outputs: 128 rows of w x m tokens, dealt to the cluster's CTAs; a warp has 32 neighbours of one token
    const Alpha alpha = F == MxFormat::kNvFp4 ? product_scale(g.x_g, g.w_g) : Alpha{1.f, 1.f};
    const uint32_t part_addr = smem_u32(part);
    uint32_t peers[kFewSplits];
#pragma unroll
    for (int s = 0; s < kFewSplits; ++s) peers[s] = s < pl.splits ? mapa_shared(part_addr, s) : 0;
    const int ykt = g.codes ? static_cast<int>(mx_scale_tiles(MxFormat::kMxFp8, g.n)) : 0;
    const int n = nt * 128 + (threadIdx.x & 127);
    float bias = 0.f;
    if (g.bias && n < g.n)
        bias = g.bias_elt == Elt::kF32 ? static_cast<const float*>(g.bias)[n]
               : g.bias_elt == Elt::kBF16 ? to_f(static_cast<const __nv_bfloat16*>(g.bias)[n])
                                          : to_f(static_cast<const __half*>(g.bias)[n]);
    const int step = pl.splits * (kFewThreads / 128);      // tokens between a thread's outputs
    constexpr int kOuts = 2;                               // ... of which so many are read together
    for (int t0 = (rank * kFewThreads + threadIdx.x) >> 7; t0 < g.m; t0 += kOuts * step) {
        float p[kOuts][kFewSplits];
#pragma unroll
        for (int o = 0; o < kOuts; ++o)
#pragma unroll
            for (int s = 0; s < kFewSplits; ++s)
                p[o][s] = (s < pl.splits && t0 + o * step < g.m) ? ld_cluster(peers[s] + ((t0 + o * step) * 128 + (threadIdx.x & 127)) * 4) : 0.f;
#pragma unroll
        for (int o = 0; o < kOuts; ++o) {
            const int t = t0 + o * step;
            if (t >= g.m) break;                           // (the same for a warp)
            float v = p[o][0];
#pragma unroll
            for (int s = 1; s < kFewSplits; ++s) v += p[o][s];
            v = fmaf(v * alpha.pre, alpha.rest, bias);
            if (g.act == 1) v = gelu_fwd(v);
            else if (g.act == 2) v = v < 0.f ? 0.f : v;    // (keeps a NaN)
            if (g.codes) {
                if (n >= g.n) v = 0.f;
                const BlockScale sc = pow2_scale<8>(__uint_as_float(__reduce_max_sync(0xffffffffu, abs_bits(v))));
                if (n < g.y_pitch)
                    static_cast<uint8_t*>(g.codes)[t * g.y_pitch + n] = static_cast<uint8_t>(cvt_e4m3x2(v * sc.inv, 0.f));
                if (lane == 0 && nt < ykt)
                    static_cast<uint8_t*>(g.scales)[scale_offset(t, n / 32, ykt)] = static_cast<uint8_t>(n < g.n ? sc.byte : 0u);
            } else if (n < g.n) {
                const int64_t at = static_cast<int64_t>(t) * g.n + n;
                if (g.out == Elt::kBF16) static_cast<__nv_bfloat16*>(g.y)[at] = __float2bfloat16_rn(v);
                else if (g.out == Elt::kF16) static_cast<__half*>(g.y)[at] = __float2half_rn(v);
                else static_cast<float*>(g.y)[at] = v;
            }
        }
    }
    if (g.codes && rank == 0 && nt < ykt)     // rows that fill the scale tile
        for (int t = g.m + threadIdx.x; t < 128; t += kFewThreads)
            *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(g.scales) + scale_offset(t, 4 * nt, ykt)) = 0;
    cluster_sync_all();      // nobody's shared memory goes while another CTA reads it
}

// Slices and shared memory of an m x n x k product; splits = 0: does not fit (x's slice is held whole).
template <MxFormat F>
FewPlan few_plan(int m, int n, int k) {
    constexpr int kAtoms = Kind<F>::kAtoms;
    FewPlan p{};
    const int tok = m <= 8 ? 8 : (m <= 16 ? 16 : 32);
    const int nts = (n + 127) / 128;
    p.ktiles = (k + Kind<F>::kElems - 1) / Kind<F>::kElems;
    // as many slices as give two CTAs an SM, at most 8 and at least one stage each
    p.splits = 1;
    while (p.splits < kFewSplits && 2 * p.splits <= p.ktiles && 2 * p.splits * nts <= 2 * num_sms()) p.splits *= 2;
    for (; p.splits <= kFewSplits; p.splits *= 2) {
        p.kt_per = (p.ktiles + p.splits - 1) / p.splits;
        const int least = std::min(p.kt_per, p.splits == kFewSplits ? 2 : 3);
        for (p.stages = std::min(p.kt_per, kFewStages); p.stages >= least; --p.stages) {
            const int64_t w = std::max(p.stages * (kWTile + kAtoms * 512), m * 512);
            const int64_t b = (w + 1023) / 1024 * 1024, sfb = b + static_cast<int64_t>(p.kt_per) * tok * kRowBytes;
            const int64_t ctl = sfb + static_cast<int64_t>(p.kt_per) * kAtoms * 512;
            p.b_off = static_cast<uint32_t>(b);
            p.sfb_off = static_cast<uint32_t>(sfb);
            p.ctl_off = static_cast<uint32_t>(ctl);
            p.smem = static_cast<uint32_t>(ctl + sizeof(FewCtl) + 1024);
            if (ctl + static_cast<int64_t>(sizeof(FewCtl)) + 1024 <= kFewSmemMax) return p;
        }
    }
    p.splits = 0;
    return p;
}

template <MxFormat F, int kTok, typename T>
cudaError_t few_launch(const MxFewArgs& a, const FewPlan& pl, cudaStream_t st) {
    const MxGemmArgs& g = a.g;
    CUtensorMap tw, sw;
    const int64_t row_bytes = (static_cast<int64_t>(g.k) * mx_bits(F) + 7) / 8;
    if (!codes_map(&tw, g.w_codes, row_bytes, g.n, g.w_pitch, 128) ||
        !scales_map(&sw, g.w_scales, g.n, static_cast<int>(mx_scale_tiles(F, g.k)), Kind<F>::kAtoms, 1))
        return cudaErrorInvalidValue;
    auto kern = mx_few_kernel<F, kTok, T>;
    static std::atomic<uint64_t> allowed{0};
    const cudaError_t e = allow_smem(kern, allowed, kFewSmemMax);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(pl.splits * ((g.n + 127) / 128));
    cfg.blockDim = dim3(kFewThreads);
    cfg.dynamicSmemBytes = pl.smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = pl.splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, tw, sw, a, pl, row_align(a.x, a.ldx * static_cast<int64_t>(sizeof(T))));
}

template <MxFormat F, typename T>
cudaError_t few_by_tokens(const MxFewArgs& a, const FewPlan& pl, cudaStream_t st) {
    if (a.g.m <= 8) return few_launch<F, 8, T>(a, pl, st);
    if (a.g.m <= 16) return few_launch<F, 16, T>(a, pl, st);
    return few_launch<F, 32, T>(a, pl, st);
}

template <MxFormat F>
cudaError_t few_by_input(const MxFewArgs& a, cudaStream_t st) {
    const FewPlan pl = few_plan<F>(a.g.m, a.g.n, a.g.k);
    if (!pl.splits) return cudaErrorInvalidValue;
    if (!a.x) return few_by_tokens<F, uint8_t>(a, pl, st);
    if (a.x_elt == Elt::kBF16) return few_by_tokens<F, __nv_bfloat16>(a, pl, st);
    if (a.x_elt == Elt::kF16) return few_by_tokens<F, __half>(a, pl, st);
    return few_by_tokens<F, float>(a, pl, st);
}

}  // namespace

// Where it beats the tiles of mx_gemm.cu (graph replays, us, few / tiles): 16-bit x, 16 tokens, 8.8 / 10.4 (nvfp4
// 4096 x 4096) and 19.0 / 22.7 (mxfp8 8192 x 8192); 32 tokens, 10.3 / 10.6 and 28.3 / 22.8: every CTA quantises its
// slice of all tokens.  x quantised before, one token: 7.1 / 8.1 and 14.6 / 30.6, but 5.2 / 3.8 (mxfp4 1536 x 384) and
// 5.9 / 5.5 (mxfp8 2048 x 1024), whose reduction is too short to cut.
bool mx_few_fits(MxFormat f, int m, int n, int k, bool quantised_x) {
    if (m > kMxFewTokens) return false;
    const int stages = (k + (f == MxFormat::kMxFp8 ? 127 : 255)) / (f == MxFormat::kMxFp8 ? 128 : 256);
    if (quantised_x ? (m > 16 || stages < 16) : (m > 16 && stages > 16)) return false;
    if (f == MxFormat::kMxFp4) return few_plan<MxFormat::kMxFp4>(m, n, k).splits > 0;
    if (f == MxFormat::kNvFp4) return few_plan<MxFormat::kNvFp4>(m, n, k).splits > 0;
    return few_plan<MxFormat::kMxFp8>(m, n, k).splits > 0;
}

cudaError_t launch_mx_few(const MxFewArgs& a, cudaStream_t st) {
    const MxGemmArgs& g = a.g;
    if (g.m <= 0 || g.m > kMxFewTokens || g.n <= 0 || g.k <= 0) return cudaErrorInvalidValue;
    int dev = 0;      // the tensor maps are encoded through the driver API, which needs a current context
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaSetDevice(dev);
    if (e != cudaSuccess) return e;
    if (g.fmt == MxFormat::kMxFp4) return few_by_input<MxFormat::kMxFp4>(a, st);
    if (g.fmt == MxFormat::kNvFp4) return few_by_input<MxFormat::kNvFp4>(a, st);
    return few_by_input<MxFormat::kMxFp8>(a, st);
}

}  // namespace mmltk
