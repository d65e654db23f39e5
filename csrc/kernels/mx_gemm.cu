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
// Persistent: warp 0 loads (TMA: codes as 128-byte swizzled boxes, scale tiles as 512-byte
// rows), warp 1 copies each stage's scales to tensor memory (tcgen05.cp, ordered before the MMAs of the
// same thread) and issues the MMAs, sixteen warps are the epilogue.  Two accumulators let it run under the
// next tile's products, and two sets of scale columns let a stage's copies run under the MMAs before
// them.  With 256 columns all of that does not fit the 512 columns of tensor memory: the accumulators
// share some, and the epilogue drains the shared ones first.
//
// Large products run on CTA pairs (cta_group::2): 256 x 256 tiles, each CTA holding its 128 rows of x
// and half of the tile's rows of w, and the scales of both (the tile's w scales are needed next to
// each CTA's accumulator).  What bounds a product of this kind is the operands' way from L2: a
// 128 x 256 tile of one CTA needs 54 KB per 512 tensor-core cycles, a pair's half 38 KB.
//
// The output leaves through tensor stores of 128-byte rows (whole lines; 32-byte sectors straight from
// registers took as long as the rest of a short product together).  The quantised output (mxfp8) needs
// no second pass: a thread has 32 consecutive columns of a row, one scale block.
//
// Few tiles and a long reduction: the CTAs of a cluster each take a slice of it, leave their partial sums in
// their (now free) stages, and after a cluster barrier each finishes a part of the columns, adding the slices in order.
//
// Measured (B200, CUDA-graph replays, x quantised before), 8192^3: mxfp8 370 to 387 us (2.9 PFLOP/s), mxfp4 195 to 197 us
// (5.6), nvfp4 222 to 234 us (4.8) in bursts of some milliseconds.  Over two seconds the power cap sets in: mxfp8 445 us
// at 1.24 GHz (2.5), mxfp4 223 at 1.49 (4.9), nvfp4 255 at 1.51 (4.3); a bf16 cuBLAS product there 1.43 PFLOP/s at
// 1.38 GHz.  The tensor pipe is busy 74 % of the cycles (4096^3 mxfp8).  nvfp4 is slower than mxfp4 by its scale copies: 12 a stage take 132
// cycles beside the MMAs' 512, 6 take 52, 3 none.  Short products are bound by issue slots: at
// 31200 x 2048 x 256 to mxfp8 (29 us; 66 MB out, 10 us) the epilogue's warps use 58 % of them, and the
// scheduler keeps a ready warp going, so the issuing warp waits for the epilogue's bursts.
//
// Every wait is bounded: on a time-out the kernel records which role gave up in a status word and
// leaves, after releasing its tensor memory.
#include "mx_mma.cuh"

namespace mmltk {

namespace {

using namespace mx;
using namespace tc;

constexpr int kEpiWarps = 16;
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kATile = 128 * kRowBytes;
constexpr int kMaxStages = 6;
constexpr int kSmemMax = 227 * 1024;

template <MxFormat F, int BN_, bool kPair, int kSize>     // kSize: bytes of an output element
struct Cfg {
    static constexpr int BN = BN_;
    static constexpr int kAtoms = Kind<F>::kAtoms;
    static constexpr int kRows = kPair ? 256 : 128;
    static constexpr int kBRows = kPair ? BN / 2 : BN;          // rows of w that a CTA holds
    static constexpr int kBTile = kBRows * kRowBytes;
    static constexpr int kSfA = kAtoms * 512;
    static constexpr int kSfB = (BN / 128) * kAtoms * 512;
    static constexpr int kStageBytes = kATile + kBTile + kSfA + kSfB;
    // staging of a warp's 32 output rows: 128-byte rows are whole lines, but the pair's long products need the
    // room for their stages
    static constexpr int kBoxBytes = BN == 256 && kPair && kSize < 4 ? 64 : 128;
    static constexpr int kBox = BN / 4 * kSize <= kBoxBytes ? BN / 4 : kBoxBytes / kSize;   // columns
    static constexpr int kRow = kBox * kSize;
    static constexpr int kStaging = 32 * kRow;
    static constexpr int kFixed = kEpiWarps * kStaging + 4 * BN * 4 + 1024 + 256;
    static constexpr int kStages =
        (kSmemMax - kFixed) / kStageBytes < kMaxStages ? (kSmemMax - kFixed) / kStageBytes : kMaxStages;
    static constexpr size_t kSmemBytes = static_cast<size_t>(kStages) * kStageBytes + kFixed;
    // tensor memory: accumulators at columns 0 and kAcc1, two sets of scales at the end
    static constexpr int kSfSet = kAtoms * 4 * (1 + BN / 128);
    static constexpr int kSfCol = 512 - 2 * kSfSet;
    static constexpr int kAcc1 = kSfCol - BN < BN ? kSfCol - BN : BN;
    static constexpr int kShared = (BN - kAcc1 + 31) / 32;      // 32-column chunks with columns of both accumulators
    static constexpr int kSharers = (kShared * 32 + BN / 4 - 1) / (BN / 4);   // column quarters with such chunks
    static_assert(kStages >= 2 && kBox % 32 == 0 && kAcc1 > 0 && kShared <= BN / 64);
};

struct __align__(8) Ctl {
    uint64_t full[kMaxStages];
    uint64_t empty[kMaxStages];
    uint64_t acc_full[2];
    uint64_t acc_empty[2];
    uint64_t shared_empty[2];     // the columns that both accumulators use have been read
    uint64_t drained;             // all MMAs of a kernel that gives up
    uint32_t tmem_base;
    int abort;
    int next_stage;               // where the loading warp stopped, for a drain
    uint32_t next_phase;
};

struct Sched {
    int m_tiles, n_tiles, ktiles, units;
    int splits, kt_per;           // slices of the reduction (the CTAs of a cluster) and their stages
    uint32_t per, magic;          // tiles of a group of 8 row tiles, and 2^32 / per
    // groups of 8 row tiles, column by column inside a group: the tiles in flight share operand rows in L2.
    // (Every role walks the tiles; plain divisions here cost the loading warp a third of a short tile's time.)
    __device__ void tile(uint32_t u, int& mt, int& nt) const {
        uint32_t g = __umulhi(u, magic);
        while (g * per > u) --g;
        while ((g + 1) * per <= u) ++g;
        const uint32_t rest = u - g * per, height = m_tiles - 8 * g;
        if (height >= 8) {
            mt = 8 * g + (rest & 7);
            nt = rest >> 3;
        } else {
            mt = 8 * g + rest % height;
            nt = rest / height;
        }
    }
};

// Staging tiles: 32 rows (lane = row) of kRow bytes in the tensor store's swizzle of that width.
template <int kRow>
__device__ __forceinline__ uint4* staged(unsigned char* buf, int row, int piece) {
    const int sw = kRow == 128 ? row & 7 : (kRow == 64 ? (row >> 1) & 3 : (row >> 2) & 1);
    return reinterpret_cast<uint4*>(buf + row * kRow) + (piece ^ sw);
}
// The staging tile may be written again: the last store from it has been read.
__device__ __forceinline__ void staging_free(int lane) {
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    __syncwarp();
}
__device__ __forceinline__ void staging_store(int lane, const CUtensorMap* map, const unsigned char* buf, int col, int row0) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) {
        asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map),
                     "r"(smem_u32(buf)), "r"(col), "r"(row0)
                     : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
}

// Output rows that are no multiple of 16 bytes, from a staging tile at (row0, col0): a lane writes 4 bytes of a row (the
// warp one row of 128 bytes or two of 64).  A 16-bit row that starts between two words is shifted by an element, its first
// and last one written alone.
template <typename O, int kRow>
__device__ __forceinline__ void copy_rows(const MxGemmArgs& g, const unsigned char* buf, int lane, int col0, int row0) {
    constexpr int kWords = kRow / 4, kPer = 32 / kWords;
    const int rows = min(32, g.m - row0), cols = min(kRow / static_cast<int>(sizeof(O)), g.n - col0);
    const int l = lane % kWords;
    auto word = [&](int r, int j) {
        const int sw = kRow == 128 ? r & 7 : (r >> 1) & 3;
        return *reinterpret_cast<const uint32_t*>(buf + r * kRow + ((((j >> 2) ^ sw) << 4) | ((j & 3) << 2)));
    };
    __syncwarp();
    O* p = static_cast<O*>(g.y) + static_cast<int64_t>(row0 + lane / kWords) * g.n + col0;
    const int64_t step = static_cast<int64_t>(kPer) * g.n;
#pragma unroll 4
    for (int r = lane / kWords; r < rows; r += kPer, p += step) {
        const uint32_t a = word(r, l);
        if constexpr (sizeof(O) == 4) {
            if (l < cols) reinterpret_cast<uint32_t*>(p)[l] = a;
        } else {
            const int odd = static_cast<int>(reinterpret_cast<uintptr_t>(p) >> 1) & 1, e = 2 * l + odd;
            const uint32_t b = word(r, min(l + 1, kWords - 1));
            const uint32_t v = odd ? __funnelshift_r(a, b, 16) : a;
            unsigned short* q = reinterpret_cast<unsigned short*>(p);
            if (e + 1 < cols) *reinterpret_cast<uint32_t*>(q + e) = v;
            else if (e < cols) q[e] = static_cast<unsigned short>(v);
            if (odd && l == 0) q[0] = static_cast<unsigned short>(a);
        }
    }
}

// ---------------------------------------------------------------- epilogue arithmetic, two columns an instruction
using f2 = unsigned long long;
__device__ __forceinline__ f2 pack2(float lo, float hi) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float2 unpack2(f2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {    // keeps a NaN
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float ex2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// GELU(x) = x Phi(x) = max(x, 0) - |x| Phi(-|x|), with Phi(-a) = exp(-a^2 / 2) Q(a).  Q(a) = erfcx(a / sqrt 2) / 2 is
// smooth and slow: a polynomial of degree 10 on [0, 6], fitted to the least maximum of exp(-a^2 / 2) |error|
// (Lawson's reweighted least squares on 4001 Chebyshev points; 6.6e-8, and 1.1e-7 with its fp32 roundings).
// One exponential and six packed multiply-adds per value; an epilogue with the erf formula's exponential and
// reciprocal per value took 15 us of the ViT's first MLP product (10400 x 1536).
template <int kPairs>
__device__ __forceinline__ void gelu2(f2* x) {
    constexpr float kQ[11] = {0.49999994f,    -0.39893651f,   0.249916792f,   -0.132513806f,    0.0611548945f,  -0.0243139397f,
                              0.00793939643f, -0.00197462994f, 0.000339739083f, -3.52078676e-05f, 1.63169466e-06f};
    f2 a[kPairs], q[kPairs];
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
        const float2 xs = unpack2(x[j]);
        a[j] = pack2(fmaxf(-fabsf(xs.x), -6.f), fmaxf(-fabsf(xs.y), -6.f));       // -min(|x|, 6)
        q[j] = pack2(kQ[10], kQ[10]);
    }
#pragma unroll
    for (int i = 9; i >= 0; --i) {
        const float c = i & 1 ? -kQ[i] : kQ[i];                                   // Q as a polynomial of -|x|
        const f2 c2 = pack2(c, c);
#pragma unroll
        for (int j = 0; j < kPairs; ++j) q[j] = fma2(q[j], a[j], c2);
    }
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
        const float2 xs = unpack2(x[j]), ts = unpack2(mul2(mul2(x[j], x[j]), pack2(-0.72134752044448170f, -0.72134752044448170f)));
        const f2 p = mul2(q[j], pack2(ex2(ts.x), ex2(ts.y)));                     // exp(-x^2 / 2) in powers of two
        x[j] = fma2(a[j], p, pack2(max_nan(xs.x, 0.f), max_nan(xs.y, 0.f)));
    }
}

// Two values to the output's type, ReLU in the conversion where it has one.
template <typename O, bool kRelu>
__device__ __forceinline__ void convert2(f2 v, uint32_t* w) {
    const float2 t = unpack2(v);
    if constexpr (std::is_same_v<O, float>) {
        w[0] = __float_as_uint(kRelu ? max_nan(t.x, 0.f) : t.x);
        w[1] = __float_as_uint(kRelu ? max_nan(t.y, 0.f) : t.y);
    } else if constexpr (std::is_same_v<O, __half>) {
        if constexpr (kRelu) asm("cvt.rn.relu.f16x2.f32 %0, %1, %2;" : "=r"(*w) : "f"(t.y), "f"(t.x));
        else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(*w) : "f"(t.y), "f"(t.x));
    } else {
        if constexpr (kRelu) asm("cvt.rn.relu.bf16x2.f32 %0, %1, %2;" : "=r"(*w) : "f"(t.y), "f"(t.x));
        else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(*w) : "f"(t.y), "f"(t.x));
    }
}

// mxfp8 output: the 32 columns at col are one scale block; codes to w, returns the scale byte.
template <bool kRelu>
__device__ __forceinline__ uint32_t quantize_chunk(const MxGemmArgs& g, f2* x, int col, uint32_t* w) {
    if (col + 32 > g.n) {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float2 t = unpack2(x[i]);
            x[i] = pack2(col + 2 * i < g.n ? t.x : 0.f, col + 2 * i + 1 < g.n ? t.y : 0.f);
        }
    }
    float m = 0.f;      // of the magnitudes, or of the positive values; keeps a NaN
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const float2 t = unpack2(x[i]);
        if constexpr (kRelu) asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(t.x), "f"(t.y));
        else asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(t.x), "f"(t.y));
    }
    const BlockScale sc = pow2_scale<8>(fabsf(m));
    const f2 inv = pack2(sc.inv, sc.inv);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 a = unpack2(mul2(x[2 * i], inv)), b = unpack2(mul2(x[2 * i + 1], inv));
        unsigned short lo, hi;
        if constexpr (kRelu) {
            asm("cvt.rn.satfinite.relu.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(a.y), "f"(a.x));
            asm("cvt.rn.satfinite.relu.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(b.y), "f"(b.x));
        } else {
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(a.y), "f"(a.x));
            asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(b.y), "f"(b.x));
        }
        w[i] = static_cast<uint32_t>(lo) | (static_cast<uint32_t>(hi) << 16);
    }
    return sc.byte;
}

// 32 accumulator columns of this thread's row on their way to registers; settled by tmem_settle
__device__ __forceinline__ void tmem_issue32(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_settle(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                   "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                   "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]),
                   "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}

// kSplit: few tiles and a long reduction.  Each CTA of a cluster multiplies a slice of it for the same 128 x 128 tile;
// the partial sums meet in shared memory, and each CTA finishes its share of the column quarters, adding the slices
// in their order.
template <MxFormat F, int BN_, bool kPair, bool kSplit, typename O, bool kQuantOut>
__global__ void __launch_bounds__(kThreads, 1)
    mx_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                   const __grid_constant__ CUtensorMap tmSA, const __grid_constant__ CUtensorMap tmSB,
                   const __grid_constant__ CUtensorMap tmY, MxGemmArgs g, Sched sch, bool tensor_store) {
    constexpr int kSize = kQuantOut ? 1 : static_cast<int>(sizeof(O));
    using C = Cfg<F, BN_, kPair, kSize>;
    using K = Kind<F>;
    constexpr int BN = C::BN, kStages = C::kStages, kAtoms = C::kAtoms;
    extern __shared__ __align__(1024) unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* tilesA = smem;
    unsigned char* tilesB = tilesA + kStages * kATile;
    unsigned char* staging = tilesB + kStages * C::kBTile;
    unsigned char* sfA = staging + kEpiWarps * C::kStaging;
    unsigned char* sfB = sfA + kStages * C::kSfA;
    float* bias_s = reinterpret_cast<float*>(sfB + kStages * C::kSfB);
    Ctl* ctl = reinterpret_cast<Ctl*>(bias_s + 4 * BN);
    // values that the compiler can see are the same in a whole warp stay in uniform registers, which is where the
    // asynchronous instructions take their operands from
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rank = kPair ? blockIdx.x & 1 : 0;
    const int slice = kSplit ? blockIdx.x % sch.splits : 0;
    const int first = kSplit ? blockIdx.x / sch.splits : (kPair ? blockIdx.x >> 1 : blockIdx.x);
    const int step = kSplit ? sch.units : (kPair ? gridDim.x >> 1 : gridDim.x);      // (kSplit: one tile a cluster)
    const int kt0 = kSplit ? slice * sch.kt_per : 0, kts = kSplit ? min(sch.kt_per, sch.ktiles - kt0) : sch.ktiles;
    static_assert(!kSplit || (BN == 128 && !kPair));

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&ctl->full[s], 1);
            mbar_init(&ctl->empty[s], 1);
        }
        // the epilogue warps of both CTAs of a pair arrive on the even CTA's barriers
        for (int b = 0; b < 2; ++b) {
            mbar_init(&ctl->acc_full[b], 1);
            mbar_init(&ctl->acc_empty[b], kEpiWarps * (kPair ? 2 : 1));
            mbar_init(&ctl->shared_empty[b], 4 * C::kSharers * (kPair ? 2 : 1));
        }
        mbar_init(&ctl->drained, 1);
        ctl->abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 0) {
        if constexpr (kPair) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl->tmem_base)),
                         "r"(512));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl->tmem_base)),
                         "r"(512));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (kPair) cluster_sync_all();   // the other CTA's barriers are initialised before anything targets them
    tc_fence_after();
    wait_previous();
    allow_next();
    constexpr uint32_t tmem = 0;                // all 512 columns are this CTA's: they start at 0

    if (warp == 0) {
        const uint32_t elected = elect_lane();
        const uint32_t sa = smem_u32(tilesA), sb = smem_u32(tilesB), pa = smem_u32(sfA), pb = smem_u32(sfB);
        const uint32_t full0 = kPair ? mapa_shared(smem_u32(&ctl->full[0]), 0) : smem_u32(&ctl->full[0]);
        int s = 0;
        uint32_t phase = 1;
        for (int u = first; u < sch.units; u += step) {
            int mt, nt;
            sch.tile(u, mt, nt);
            const int rt = kPair ? 2 * mt + rank : mt;      // this CTA's tile of 128 rows
            for (int kt = kt0; kt < kt0 + kts; ++kt) {
                // (the second look: so that both loading warps of a pair that gives up stop at the same stage)
                if (!__all_sync(0xffffffffu, mbar_wait(&ctl->empty[s], phase, &ctl->abort)) &&
                    !__all_sync(0xffffffffu, mbar_try_wait(&ctl->empty[s], phase))) {
                    if (elected) {
                        ctl->abort = 1;
                        atomicCAS(g.status, 0, 1);
                    }
                    goto producer_done;
                }
                // boxes past an extent are zero-filled and count in full
                if (rank == 0 && elected) mbar_expect_tx(&ctl->full[s], C::kStageBytes * (kPair ? 2 : 1));
                const uint32_t bar = full0 + 8 * s;
                load_2d<kPair>(elected, &tmA, bar, sa + s * kATile, kt * kRowBytes, rt * 128);
                load_2d<kPair>(elected, &tmB, bar, sb + s * C::kBTile, kt * kRowBytes, nt * BN + rank * C::kBRows);
                load_3d<kPair>(elected, &tmSA, bar, pa + s * C::kSfA, 0, kt * kAtoms, rt);
                load_3d<kPair>(elected, &tmSB, bar, pb + s * C::kSfB, 0, kt * kAtoms, nt * (BN / 128));
                if (++s == kStages) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
    producer_done:
        if (elected) {
            ctl->next_stage = s;
            ctl->next_phase = phase;
        }
        if constexpr (kSplit) cluster_sync_all();
    } else if (warp == 1) {
        if (rank == 0) {
            const uint32_t elected = elect_lane();
            constexpr uint32_t idesc = K::kDesc | (static_cast<uint32_t>(BN >> 3) << 17) |
                                       (static_cast<uint32_t>(C::kRows >> 4) << 24);
            const uint32_t a0 = operand_lo(smem_u32(tilesA)), b0 = operand_lo(smem_u32(tilesB));
            const uint32_t pa0 = smem_u32(sfA) >> 4, pb0 = smem_u32(sfB) >> 4;
            const uint32_t empty0 = smem_u32(&ctl->empty[0]), accf0 = smem_u32(&ctl->acc_full[0]);
            // the other CTA's barriers (shared::cluster addresses run on like the shared ones)
            const uint32_t empty1 = kPair ? mapa_shared(empty0, 1) : 0, accf1 = kPair ? mapa_shared(accf0, 1) : 0;
            int local = 0, s = 0;
            uint32_t phase = 0, set = 0, ready = 0;
            for (int u = first; u < sch.units; u += step, ++local) {
                const int buf = local & 1;
                // the accumulator was read two tiles ago, the columns it shares in the last one (both asked for together)
                const uint32_t phase_a = ((local >> 1) & 1) ^ 1, phase_s = ((local - 1) >> 1) & 1;
                const bool shared = C::kShared && local > 0;
                const uint32_t free_s = shared ? mbar_try_wait_cluster(&ctl->shared_empty[buf ^ 1], phase_s) : 1u;
                const uint32_t free_a = mbar_try_wait_cluster(&ctl->acc_empty[buf], phase_a);
                bool ok = true;
                if (!__all_sync(0xffffffffu, free_a & free_s)) {
                    ok = mbar_wait_cluster(&ctl->acc_empty[buf], phase_a, &ctl->abort);
                    if (shared) ok = ok && mbar_wait_cluster(&ctl->shared_empty[buf ^ 1], phase_s, &ctl->abort);
                    ok = __all_sync(0xffffffffu, ok);
                }
                tc_fence_after();
                const uint32_t acc = tmem + buf * C::kAcc1;
                int left = kSplit ? min(g.k - kt0 * K::kElems, kts * K::kElems) : g.k;
                uint32_t more = 0;
                for (; ok && left > 0; left -= K::kElems) {
                    if (!ready) ok = __all_sync(0xffffffffu, mbar_wait(&ctl->full[s], phase, &ctl->abort, g.wait_limit));
                    if (!ok) break;
                    tc_fence_after();
                    // ask for the next stage now and look at the answer after this one's MMAs: a wait costs 170
                    // cycles even on a full stage, and the tensor core's queue is too short to cover them
                    const int s1 = s + 1 == kStages ? 0 : s + 1;
                    const uint32_t phase1 = s + 1 == kStages ? phase ^ 1 : phase;
                    const uint32_t seen = mbar_test(&ctl->full[s1], phase1);
                    const uint32_t a = a0 + s * (kATile >> 4), b = b0 + s * (C::kBTile >> 4);
                    const uint32_t pa = pa0 + s * (C::kSfA >> 4), pb = pb0 + s * (C::kSfB >> 4);
                    // scale tile j: x's at columns tsa + 4 j; w's row tiles side by side for each j
                    const uint32_t tsa = tmem + C::kSfCol + set, tsb = tsa + 4 * kAtoms;
#pragma unroll
                    for (int j = 0; j < kAtoms; ++j) {
                        copy_scales<kPair>(elected, tsa + 4 * j, pa + j * 32);
#pragma unroll
                        for (int r = 0; r < BN / 128; ++r)
                            copy_scales<kPair>(elected, tsb + (BN / 128) * 4 * j + 4 * r, pb + (r * kAtoms + j) * 32);
                    }
                    // MMAs that would only see padding are left out
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        if (kk * (K::kElems / 4) < left) {
                            const int j = kk * kAtoms / 4;
                            const uint32_t id = F == MxFormat::kNvFp4 ? 0u : (F == MxFormat::kMxFp4 ? (kk & 1) * 2u : kk);
                            mma_block<F, kPair>(elected, acc, a + 2 * kk, b + 2 * kk, idesc | (id << 4) | (id << 29),
                                                tsa + 4 * j, tsb + (BN / 128) * 4 * j, more);
                            more = 1;
                        }
                    }
                    if constexpr (kPair) {
                        commit<true>(elected, empty0 + 8 * s);
                        commit<true>(elected, empty1 + 8 * s);
                    } else {
                        commit<false>(elected, empty0 + 8 * s);
                    }
                    set ^= C::kSfSet;
                    s = s1;
                    phase = phase1;
                    ready = __all_sync(0xffffffffu, seen);
                }
                if (!ok) {
                    // the MMAs under way end, and their stages are free, before anybody hears of it
                    commit<kPair>(elected, smem_u32(&ctl->drained));
                    mbar_drain(&ctl->drained, 0, drain_deadline());
                    __syncwarp();
                    if (elected) {
                        ctl->abort = 1;
                        if constexpr (kPair)      // the other CTA's roles wait for this one's barriers
                            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(mapa_shared(smem_u32(&ctl->abort), 1)), "r"(1)
                                         : "memory");
                        atomicCAS(g.status, 0, 2);
                    }
                    break;
                }
                if constexpr (kPair) {
                    commit<true>(elected, accf0 + 8 * buf);
                    commit<true>(elected, accf1 + 8 * buf);
                } else {
                    commit<false>(elected, accf0 + 8 * buf);
                }
            }
        }
        if constexpr (kSplit) cluster_sync_all();
    } else {
        // sixteen warps (four a scheduler hide the latencies of a chunk): lane quarter q, column quarter part
        const int q = warp & 3, part = (warp - 2) >> 2;
        constexpr int kCols = BN / 4, kChunks = kCols / 32;
        unsigned char* buf_s = staging + (warp - 2) * C::kStaging;
        constexpr int kBox = C::kBox, kRow = C::kRow, kPieces = 32 * kSize / 16;
        float* bias_w = bias_s + (warp - 2) * kCols;
        const Alpha alpha = F == MxFormat::kNvFp4 ? product_scale(g.x_g, g.w_g) : Alpha{1.f, 1.f};
        const int ykt = kQuantOut ? static_cast<int>(mx_scale_tiles(MxFormat::kMxFp8, g.n)) : 0;
        auto bias_at = [&](int col) {
            if (!g.bias || col >= g.n) return 0.f;
            return g.bias_elt == Elt::kF32 ? static_cast<const float*>(g.bias)[col]
                   : g.bias_elt == Elt::kBF16 ? to_f(static_cast<const __nv_bfloat16*>(g.bias)[col])
                                              : to_f(static_cast<const __half*>(g.bias)[col]);
        };
        auto flush = [&](int col, int row0) {      // the staging tile's columns from col on
            if constexpr (kQuantOut) {
                staging_store(lane, &tmY, buf_s, col, row0);
            } else {
                if (tensor_store) staging_store(lane, &tmY, buf_s, col, row0);
                else copy_rows<O, kRow>(g, buf_s, lane, col, row0);
            }
        };
        int mt = 0, nt = 0, mt_next = 0, nt_next = 0;
        float bias_r[kChunks];
        if (first < sch.units) {
            sch.tile(first, mt_next, nt_next);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) bias_r[c] = bias_at(nt_next * BN + part * kCols + 32 * c + lane);
        }
        int local = 0;
        for (int u = first; u < sch.units; u += step, ++local) {
            mt = mt_next;
            nt = nt_next;
            const int row0 = (kPair ? 2 * mt + rank : mt) * 128 + 32 * q, col0 = nt * BN + part * kCols;
            // this warp's columns of the bias; the next tile's are on their way meanwhile
            __syncwarp();
#pragma unroll
            for (int c = 0; c < kChunks; ++c) bias_w[32 * c + lane] = bias_r[c];
            __syncwarp();
            if (u + step < sch.units) {
                sch.tile(u + step, mt_next, nt_next);
#pragma unroll
                for (int c = 0; c < kChunks; ++c) bias_r[c] = bias_at(nt_next * BN + part * kCols + 32 * c + lane);
            }
            const int buf = local & 1;
            if (!__all_sync(0xffffffffu, mbar_wait(&ctl->acc_full[buf], (local >> 1) & 1, &ctl->abort))) {
                if (lane == 0) atomicCAS(g.status, 0, 3);
                ctl->abort = 1;
                if constexpr (kSplit) cluster_sync_all();
                break;
            }
            tc_fence_after();
            const uint32_t acc = tmem + buf * C::kAcc1 + (static_cast<uint32_t>(32 * q) << 16) + part * kCols;
            // chunks with columns of both accumulators (the first one's last, the second one's first) come first
            const int mine = buf ? min(kChunks, C::kShared - part * kChunks)
                                 : min(kChunks, C::kShared - (3 - part) * kChunks);     // how many, if positive
            uint32_t bytes = 0, freed = 0;
            bool owner = true;
#pragma unroll
            for (int i = 0; i < kChunks; ++i) {
                const int c = buf ? i : kChunks - 1 - i;
                const int col = col0 + 32 * c;
                uint32_t v[32];
                tmem_issue32(acc + 32 * c, v);
                tmem_settle(v);
                if ((C::kShared && mine == i + 1) || i == kChunks - 1) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        if (C::kShared && mine == i + 1) {
                            if constexpr (kPair) mbar_arrive_remote(mapa_shared(smem_u32(&ctl->shared_empty[buf]), 0));
                            else mbar_arrive(&ctl->shared_empty[buf]);
                        }
                        if (i == kChunks - 1) {
                            if constexpr (kPair) mbar_arrive_remote(mapa_shared(smem_u32(&ctl->acc_empty[buf]), 0));
                            else mbar_arrive(&ctl->acc_empty[buf]);
                        }
                    }
                }
                if constexpr (kSplit) {
                    // every operand stage has been used: their room takes the partial sums
                    const uint32_t at = smem_u32(tilesA) + (part * 4 + q) * 4096 + lane * 16;
                    owner = (part & (sch.splits - 1)) == slice;
                    if (!owner) {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + j * 512), "r"(v[4 * j]),
                                         "r"(v[4 * j + 1]), "r"(v[4 * j + 2]), "r"(v[4 * j + 3])
                                         : "memory");
                    }
                    cluster_sync_all();
                    if (!owner) continue;
                    float sum[32];
                    for (int s = 0; s < sch.splits; ++s) {
                        const uint32_t from = mapa_shared(at, s);
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            uint4 t = make_uint4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                            if (s != slice)
                                asm volatile("ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [%4];"
                                             : "=r"(t.x), "=r"(t.y), "=r"(t.z), "=r"(t.w)
                                             : "r"(from + j * 512));
                            const float4 f = make_float4(__uint_as_float(t.x), __uint_as_float(t.y), __uint_as_float(t.z),
                                                         __uint_as_float(t.w));
                            sum[4 * j] = s ? sum[4 * j] + f.x : f.x;
                            sum[4 * j + 1] = s ? sum[4 * j + 1] + f.y : f.y;
                            sum[4 * j + 2] = s ? sum[4 * j + 2] + f.z : f.z;
                            sum[4 * j + 3] = s ? sum[4 * j + 3] + f.w : f.w;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(sum[j]);
                }
                if (col >= g.n || row0 >= g.m) continue;       // warp-uniform
                if (F == MxFormat::kNvFp4 && alpha.pre != 1.f) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = __float_as_uint(__uint_as_float(v[j]) * alpha.pre);
                }
                f2 x[16];
                const f2 alpha2 = pack2(alpha.rest, alpha.rest);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const ulonglong2 b = reinterpret_cast<const ulonglong2*>(bias_w + 32 * c)[j];
                    x[2 * j] = fma2(pack2(__uint_as_float(v[4 * j]), __uint_as_float(v[4 * j + 1])), alpha2, b.x);
                    x[2 * j + 1] = fma2(pack2(__uint_as_float(v[4 * j + 2]), __uint_as_float(v[4 * j + 3])), alpha2, b.y);
                }
                if (g.act == 1) {
#pragma unroll
                    for (int j = 0; j < 16; j += 4) gelu2<4>(x + j);
                }
                uint32_t w[8 * kSize];
                if constexpr (kQuantOut) {
                    const uint32_t byte = g.act == 2 ? quantize_chunk<true>(g, x, col, w) : quantize_chunk<false>(g, x, col, w);
                    if (row0 + lane < g.m) bytes |= byte << (8 * c);
                } else if (g.act == 2) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) convert2<O, true>(x[j], w + j * kSize / 2);
                } else {
#pragma unroll
                    for (int j = 0; j < 16; ++j) convert2<O, false>(x[j], w + j * kSize / 2);
                }
                if (freed == 0 || kBox == 32) {
                    staging_free(lane);
                    freed = 1;
                }
#pragma unroll
                for (int j = 0; j < kPieces; ++j)
                    *staged<kRow>(buf_s, lane, (kBox == 32 ? 0 : c * kPieces) + j) =
                        make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
                if (kBox == 32) flush(col, row0);
            }
            if (kBox > 32 && owner && col0 < g.n && row0 < g.m) flush(col0, row0);
            if constexpr (kQuantOut) {
                // scale bytes of this row's blocks: one or two neighbours; zero past m and n
                if (owner && row0 / 128 < (g.m + 127) / 128 && col0 / 128 < ykt) {
                    uint8_t* p = static_cast<uint8_t*>(g.scales) + scale_offset(row0 + lane, col0 / 32, ykt);
                    if constexpr (kChunks == 2) *reinterpret_cast<uint16_t*>(p) = static_cast<uint16_t>(bytes);
                    else *p = static_cast<uint8_t>(bytes);
                }
            }
        }
        if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0 && rank == 0 && ctl->abort) {
        // loads that nobody waited for (a pair's count on the even CTA's barriers): the last of each stage, which is of
        // this turn of the ring below next_stage and of the one before from there on
        const unsigned long long deadline = drain_deadline();
        for (int i = 0; i < kStages; ++i)
            mbar_drain(&ctl->full[i], i < ctl->next_stage ? ctl->next_phase ^ 1 : ctl->next_phase, deadline);
        __syncwarp();
    }
    // no CTA leaves while the pair's MMAs, or the cluster's sums, may still read its shared memory
    if constexpr (kPair || kSplit) cluster_sync_all();
    if (warp == 0) {
        tc_fence_after();
        if constexpr (kPair)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// Output: boxes of 32 rows x box columns in the swizzle of their width; stores past the extents are clipped.
bool out_map(CUtensorMap* map, void* p, Elt e, bool quant, int64_t cols, int64_t rows, int64_t pitch, int box_cols) {
    auto fn = encode_fn();
    if (!fn) return false;
    const CUtensorMapDataType dt = quant ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                   : e == Elt::kF32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : e == Elt::kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                    : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const int row = box_cols * (quant ? 1 : e == Elt::kF32 ? 4 : 2);
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(pitch)};
    cuuint32_t box[2] = {static_cast<cuuint32_t>(box_cols), 32u}, es[2] = {1, 1};
    return fn(map, dt, 2, p, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
              row == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : (row == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_32B),
              CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <MxFormat F, int BN, bool kPair, bool kSplit, typename O, bool kQ>
cudaError_t launch(const MxGemmArgs& g, int splits, cudaStream_t st) {
    using C = Cfg<F, BN, kPair, kQ ? 1 : static_cast<int>(sizeof(O))>;
    CUtensorMap ta, tb, sa, sb;
    const int64_t row_bytes = (static_cast<int64_t>(g.k) * mx_bits(F) + 7) / 8;
    const int kt = static_cast<int>(mx_scale_tiles(F, g.k));
    if (!codes_map(&ta, g.x_codes, row_bytes, g.m, g.x_pitch, 128) ||
        !codes_map(&tb, g.w_codes, row_bytes, g.n, g.w_pitch, C::kBRows) ||
        !scales_map(&sa, g.x_scales, g.m, kt, C::kAtoms, 1) ||
        !scales_map(&sb, g.w_scales, g.n, kt, C::kAtoms, BN / 128))
        return cudaErrorInvalidValue;
    Sched sch;
    sch.m_tiles = (g.m + C::kRows - 1) / C::kRows;
    sch.n_tiles = (g.n + BN - 1) / BN;
    sch.ktiles = (g.k + Kind<F>::kElems - 1) / Kind<F>::kElems;
    sch.units = sch.m_tiles * sch.n_tiles;
    sch.splits = splits;
    sch.kt_per = (sch.ktiles + splits - 1) / splits;
    sch.per = 8u * sch.n_tiles;
    sch.magic = static_cast<uint32_t>((uint64_t(1) << 32) / sch.per);
    const bool tensor_store = kQ || (g.y_pitch % 16 == 0 && reinterpret_cast<uintptr_t>(g.y) % 16 == 0);
    CUtensorMap ty{};
    if (tensor_store && !out_map(&ty, kQ ? g.codes : g.y, g.out, kQ, kQ ? g.y_pitch : g.n, g.m, g.y_pitch, C::kBox))
        return cudaErrorInvalidValue;
    auto kern = mx_gemm_kernel<F, BN, kPair, kSplit, O, kQ>;
    static std::atomic<uint64_t> allowed{0};
    const cudaError_t e = allow_smem(kern, allowed, static_cast<int>(C::kSmemBytes));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(kSplit ? sch.units * splits : kPair ? 2 * std::min(sch.units, num_sms() / 2) : std::min(sch.units, num_sms()));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = C::kSmemBytes;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = kSplit ? splits : 2;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = kPair || kSplit ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, ta, tb, sa, sb, ty, g, sch, tensor_store);
}

template <MxFormat F, int BN, bool kPair, bool kSplit>
cudaError_t by_output(const MxGemmArgs& g, cudaStream_t st, int splits = 1) {
    if (g.codes) return launch<F, BN, kPair, kSplit, float, true>(g, splits, st);
    if (g.out == Elt::kBF16) return launch<F, BN, kPair, kSplit, __nv_bfloat16, false>(g, splits, st);
    if (g.out == Elt::kF16) return launch<F, BN, kPair, kSplit, __half, false>(g, splits, st);
    return launch<F, BN, kPair, kSplit, float, false>(g, splits, st);
}

template <MxFormat F>
cudaError_t by_tile(const MxGemmArgs& g, cudaStream_t st) {
    // Pairs where the reduction is long (8 stages) and the pairs get two tiles each: at 8192^3, both timed in turn at the
    // power cap, they take 392 us where 128 x 256 tiles of single CTAs take 462 (mxfp8) and 224 against 318 (nvfp4); at K = 256 they lose (31200 x 2048:
    // 45 us against 30), each tile's hand-overs crossing the pair.  Else the width whose waves cost less, a
    // 256-column tile counting 1.75 of a 128-column one (31200 x 2048 x 256: 33.4 and 30.0; 10400 x 1536 x 384: 18.3
    // and 19.6; 512 x 4096 x 4096: 9.9 and 13.6).
    const int64_t sms = num_sms(), rt = (g.m + 127) / 128;
    const int64_t pairs = (rt + 1) / 2 * ((g.n + 255) / 256);
    if (g.k >= 8 * Kind<F>::kElems && pairs >= sms) return by_output<F, 256, true, false>(g, st);
    const int64_t w128 = (rt * ((g.n + 127) / 128) + sms - 1) / sms, w256 = (rt * ((g.n + 255) / 256) + sms - 1) / sms;
    if (7 * w256 < 4 * w128) return by_output<F, 256, false, false>(g, st);
    const int64_t tiles = rt * ((g.n + 127) / 128);
    const int ktiles = (g.k + Kind<F>::kElems - 1) / Kind<F>::kElems;
    // Slices of a long reduction where the tiles leave SMs idle: the cluster costs 3 us and a stage 0.33 us, so from 24
    // stages on (one / two / four slices: mxfp8 93 x 301 x 4641 17.7 / 14.4 / 12.8, 48 x 8192 x 8192 20.7 / 16.0 / -,
    // mxfp4 512 x 1024 x 8192 12.6 / 11.0 / 11.0; nvfp4 128 x 4096 x 4096, 16 stages, 8.5 / 9.0 / 9.7).
    for (int splits = 4; splits > 1 && ktiles >= 24; splits /= 2) {
        const int per = (ktiles + splits - 1) / splits;
        if (tiles * splits <= sms && (splits - 1) * per < ktiles) return by_output<F, 128, false, true>(g, st, splits);
    }
    return by_output<F, 128, false, false>(g, st);
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
