// Kernel arguments and launch functions of the feature operators (group norm, dropout, rotary
// positions).  The launch functions only enqueue; ta_api_features.cuh checks the arguments first.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace ta {

enum { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3 };

struct GnArgs {
    const void *x, *weight, *bias, *dy;
    void *y, *dx, *dweight, *dbias;
    float *mean, *rstd;             // [n, groups]
    float2 *part, *channel_part;    // scratch, see scratch_group_norm_*()
    long long n, rows;
    int channels, groups, cpg;      // cpg = channels / groups
    int param_code, act;
    int wide_params;                // weight and bias: float32 on 16-byte boundaries
    float eps;
    int sm_count;
};

// scratch of a forward (backward = false) or backward call, bytes
size_t scratch_group_norm_f32(const GnArgs &a, bool backward);
size_t scratch_group_norm_f16(const GnArgs &a, bool backward);
size_t scratch_group_norm_bf16(const GnArgs &a, bool backward);
cudaError_t launch_group_norm_f32(const GnArgs &a, bool backward, cudaStream_t stream);
cudaError_t launch_group_norm_f16(const GnArgs &a, bool backward, cudaStream_t stream);
cudaError_t launch_group_norm_bf16(const GnArgs &a, bool backward, cudaStream_t stream);

// n / d for 32-bit n by a multiplication (Granlund and Montgomery, "Division by invariant integers using multiplication", 1994)
struct FastDiv {
    uint32_t d, m, s1, s2;
};
inline FastDiv fast_div_of(uint32_t d)
{
    uint32_t l = 0;
    while (l < 32 && (1ull << l) < d) ++l;
    FastDiv f;
    f.d = d;
    f.m = (uint32_t)((((1ull << l) - d) << 32) / d + 1);
    f.s1 = l < 1 ? l : 1;
    f.s2 = l < 1 ? 0 : l - 1;
    return f;
}

struct DropoutArgs {
    const void *x, *residual;
    void *y;
    const uint64_t *seed_ptr;
    uint64_t seed;
    long long numel;
    long long size[4], mstride[4];  // merged dimensions, outermost first, padded in front with size 1
    FastDiv div[4];                 // of size[], where numel is below 2^32
    uint32_t offset, thr_hi, thr_lo; // keep: (16-bit number, 16-bit refinement) >= (thr_hi, thr_lo)
    int drop_all;                   // the threshold is 2^32: above every number
    float scale;
    int sm_count;
};
cudaError_t launch_dropout(const DropoutArgs &a, int dtype, cudaStream_t stream);

constexpr int kRotaryMaxPairs = 256;
struct RotaryArgs {
    const void *q, *k;
    void *q_out, *k_out;
    long long qs[3], ks[3], qos[3], kos[3];      // element strides of sample, token, head
    long long n, tokens;
    int prefix, q_heads, k_heads, dim, axes, pairs;
    int halves;                                  // 1: pair j = elements (j, j + pairs); 0: (2j, 2j + 1)
    int inverse;
    int pos_kind;                                // 0 grid, 1 int64, 2 float32, 3 int32
    const void *positions;
    long long pos_s[3];                          // element strides of sample, token, axis
    int grid[3];
    FastDiv grid_div[3], token_div;              // token_div: of tokens
    float patch;
    const float *top, *left;
    const uint8_t *flip;
    int sm_count;
    float freq_hi[kRotaryMaxPairs], freq_lo[kRotaryMaxPairs];   // turns per unit of position
    int axis_end[3];                             // pair j belongs to the first axis a with j < axis_end[a]
};
cudaError_t launch_rotary(const RotaryArgs &a, int dtype, cudaStream_t stream);

}  // namespace ta
