// Launchers of the microscaled formats, their products and the RMS norm (raw pointers, no torch).
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace mmltk {

enum class MxFormat : int { kMxFp4 = 0, kNvFp4 = 1, kMxFp8 = 2 };
enum class Elt : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

constexpr int mx_block(MxFormat f) { return f == MxFormat::kNvFp4 ? 16 : 32; }
constexpr int mx_bits(MxFormat f) { return f == MxFormat::kMxFp8 ? 8 : 4; }
// bytes of a row of codes (padded to 16) and scale tiles along a row
constexpr int64_t mx_pitch(MxFormat f, int64_t dim) { return ((dim * mx_bits(f) + 7) / 8 + 15) / 16 * 16; }
constexpr int64_t mx_scale_tiles(MxFormat f, int64_t dim) { return (dim + 4 * mx_block(f) - 1) / (4 * mx_block(f)); }

// x [rows, dim] (row pitch ld) -> codes [rows, mx_pitch], scales [ceil(rows / 128), mx_scale_tiles, 512].
// nvfp4: g (fp32 [1], null: 1) is the tensor's scale; with amax (uint32 [kMxAmaxParts], work space) g is an output,
// found first.
constexpr int kMxAmaxParts = 512;
cudaError_t launch_mx_quantize(Elt et, MxFormat f, const void* x, int64_t ld, int64_t rows, int64_t dim, void* codes,
                               void* scales, float* g, uint32_t* amax, cudaStream_t st);
cudaError_t launch_mx_dequantize(Elt et, MxFormat f, const void* codes, const void* scales, const float* g,
                                 int64_t rows, int64_t dim, void* out, cudaStream_t st);

constexpr int kMxWaitLimit = 1 << 22;

// ---------------------------------------------------------------- RMS norm
constexpr int kRmsMaxDim = 16384;

struct RmsFwdArgs {
    const void* x;
    const void* res;      // optional: the norm reads round(x + res), stored to h
    const void* w;        // [dim], x's type or fp32, 16-byte aligned
    void* y;              // [rows, dim] of x's type (contiguous), or null with codes
    void* h;              // [rows, dim], with res
    float* rstd;          // optional [rows]
    void* codes;          // quantised output instead of y
    void* scales;
    const float* g;       // nvfp4
    int64_t rows, ldx, ldr;
    int dim;
    float eps;
    bool w_f32;
    MxFormat fmt;
};
cudaError_t launch_rms_fwd(Elt et, const RmsFwdArgs& a, cudaStream_t st);

struct RmsBwdArgs {
    const void* gy;       // gradient of y
    const void* gh;       // optional gradient of h
    const void* h;        // what the norm read
    const void* w;
    const float* rstd;
    void* gx;
    void* gw;             // [dim] of w's type
    float* partial;       // [rms_bwd_partials(rows), rms_partial_pitch(dim)] work space, null: no gw
    int* status;          // set when a bounded wait gave up
    int64_t rows, ldgy, ldgh, ldh;
    int dim;
    int wait_limit;       // tries of a wait for loaded data
    bool w_f32;
};
constexpr int rms_partial_pitch(int dim) { return (dim + 7) / 8 * 8; }
int rms_bwd_partials(int64_t rows);
cudaError_t launch_rms_bwd(Elt et, const RmsBwdArgs& a, cudaStream_t st);

// ---------------------------------------------------------------- product
struct MxGemmArgs {
    const void* x_codes;      // [m, pitch]
    const void* x_scales;
    const float* x_g;         // nvfp4: tensor scales (null: 1)
    const void* w_codes;      // [n, pitch]
    const void* w_scales;
    const float* w_g;
    const void* bias;         // optional [n]
    void* y;                  // [m, n] contiguous, or null with codes
    void* codes;              // mxfp8 output
    void* scales;
    int* status;
    int64_t x_pitch, w_pitch, y_pitch;   // bytes of a row
    int m, n, k;
    int wait_limit;           // tries of a wait for loaded data
    Elt out, bias_elt;
    int act;                  // 0 none, 1 GELU, 2 ReLU
    MxFormat fmt;
};
cudaError_t launch_mx_gemm(const MxGemmArgs& a, cudaStream_t st);

// Few tokens (where mx_few_fits says so): one launch that also quantises x (x != null).
constexpr int kMxFewTokens = 32;
struct MxFewArgs {
    MxGemmArgs g;
    const void* x;            // [m, k] (row pitch ldx elements) of type x_elt; null: g.x_codes / g.x_scales
    int64_t ldx;
    Elt x_elt;
};
bool mx_few_fits(MxFormat f, int m, int n, int k, bool quantised_x);
cudaError_t launch_mx_few(const MxFewArgs& a, cudaStream_t st);

}  // namespace mmltk
