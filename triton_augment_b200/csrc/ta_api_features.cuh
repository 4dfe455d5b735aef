// Entry points of the feature operators: argument checks and launches (included by ta_api.cu).
#pragma once

#include "ta_features.h"

namespace ta {

static int feature_bytes(int dtype) { return dtype == TA_B200_F32 ? 4 : dtype == TA_B200_F16 || dtype == TA_B200_BF16 ? 2 : 0; }

// ----------------------------------------------------------------------------- group norm
static int group_norm_args(const ta_b200_group_norm_params *p, bool backward, GnArgs &a)
{
    if (!p) return fail(TA_B200_ERR_NULL, "params is NULL");
    if (p->struct_size != sizeof(ta_b200_group_norm_params))
        return fail(TA_B200_ERR_SHAPE, "struct_size %u is not %zu (ABI mismatch)", p->struct_size, sizeof(ta_b200_group_norm_params));
    if (!feature_bytes(p->dtype)) return fail(TA_B200_ERR_DTYPE, "dtype %d", p->dtype);
    if ((p->weight || p->bias || p->dweight || p->dbias) && !feature_bytes(p->param_dtype))
        return fail(TA_B200_ERR_DTYPE, "param_dtype %d", p->param_dtype);
    if (p->activation < TA_B200_ACT_NONE || p->activation > TA_B200_ACT_GELU)
        return fail(TA_B200_ERR_UNSUPPORTED, "activation %d", p->activation);
    if (p->n < 0 || p->rows < 0 || p->channels <= 0 || p->groups <= 0 || p->channels % p->groups != 0)
        return fail(TA_B200_ERR_SHAPE, "bad sizes n=%lld rows=%lld channels=%d groups=%d (channels must be a multiple of groups)",
                    (long long)p->n, (long long)p->rows, p->channels, p->groups);
    if (!(p->eps >= 0.0f)) return fail(TA_B200_ERR_SHAPE, "eps must not be negative");
    if (p->n >= (1 << 22) || p->rows >= (1LL << 31) || p->channels > (1 << 20) || (double)p->n * p->rows * p->channels >= 4398046511104.0)
        return fail(TA_B200_ERR_TOO_LARGE, "at most 2^22 samples, 2^31 rows, 2^20 channels and 2^42 elements per call");
    const bool empty = p->n == 0 || p->rows == 0;
    if (!empty && (!p->x || (backward ? !p->dy || !p->mean || !p->rstd : !p->y || !p->mean || !p->rstd)))
        return fail(TA_B200_ERR_NULL, "x, mean, rstd and y (forward) or dy (backward) are required");
    memset(&a, 0, sizeof(a));
    a.x = p->x; a.weight = p->weight; a.bias = p->bias;
    a.mean = p->mean; a.rstd = p->rstd;
    if (backward) { a.dy = p->dy; a.dx = p->dx; a.dweight = p->dweight; a.dbias = p->dbias; }
    else a.y = p->y;
    a.part = (float2 *)p->scratch;
    a.n = p->n; a.rows = p->rows; a.channels = p->channels; a.groups = p->groups; a.cpg = p->channels / p->groups;
    a.param_code = p->param_dtype; a.act = p->activation; a.eps = p->eps;
    a.wide_params = p->param_dtype == TA_B200_F32 && (((uintptr_t)p->weight | (uintptr_t)p->bias) % 16) == 0;
    return TA_B200_OK;
}

static size_t group_norm_scratch(int dtype, const GnArgs &a, bool backward)
{
    return dtype == TA_B200_F32 ? scratch_group_norm_f32(a, backward) : dtype == TA_B200_F16 ? scratch_group_norm_f16(a, backward)
                                                                                           : scratch_group_norm_bf16(a, backward);
}

static int group_norm(const ta_b200_group_norm_params *p, bool backward, cudaStream_t stream)
{
    GnArgs a;
    int rc = group_norm_args(p, backward, a);
    if (rc != TA_B200_OK) return rc;
    const size_t es = feature_bytes(p->dtype), pb = feature_bytes(p->param_dtype);
    if (((uintptr_t)p->x | (uintptr_t)p->y | (uintptr_t)p->dy | (uintptr_t)p->dx) % es || ((uintptr_t)p->mean | (uintptr_t)p->rstd) % 4 ||
        (pb && ((uintptr_t)p->weight | (uintptr_t)p->bias | (uintptr_t)p->dweight | (uintptr_t)p->dbias) % pb))
        return fail(TA_B200_ERR_UNSUPPORTED, "tensors must be aligned to their elements");
    if (a.n == 0 || a.rows == 0) {
        // no element: the parameters' gradients are zero
        for (void *g : {a.dweight, a.dbias})
            if (g) {
                cudaError_t e = cudaMemsetAsync(g, 0, pb * a.channels, stream);
                if (e != cudaSuccess) return cuda_fail(e, "cudaMemsetAsync(group_norm gradients)");
            }
        return TA_B200_OK;
    }
    DeviceState *s = nullptr;
    rc = current_device(&s, nullptr);
    if (rc != TA_B200_OK) return rc;
    a.sm_count = s->sm_count;
    const size_t need = group_norm_scratch(p->dtype, a, backward);
    if (need > 0 && (!p->scratch || p->scratch_bytes < need || (uintptr_t)p->scratch % 16))
        return fail(TA_B200_ERR_SCRATCH, "scratch must be 16-byte aligned and hold %zu bytes", need);
    cudaError_t e = p->dtype == TA_B200_F32 ? launch_group_norm_f32(a, backward, stream)
                  : p->dtype == TA_B200_F16 ? launch_group_norm_f16(a, backward, stream)
                                            : launch_group_norm_bf16(a, backward, stream);
    if (e != cudaSuccess) return cuda_fail(e, "launch(group_norm)");
    return TA_B200_OK;
}

// ----------------------------------------------------------------------------- dropout
static int dropout(const ta_b200_dropout_params *p, cudaStream_t stream)
{
    if (!p) return fail(TA_B200_ERR_NULL, "params is NULL");
    if (p->struct_size != sizeof(ta_b200_dropout_params))
        return fail(TA_B200_ERR_SHAPE, "struct_size %u is not %zu (ABI mismatch)", p->struct_size, sizeof(ta_b200_dropout_params));
    const size_t es = feature_bytes(p->dtype);
    if (!es) return fail(TA_B200_ERR_DTYPE, "dtype %d", p->dtype);
    if (!(p->p >= 0.0 && p->p <= 1.0)) return fail(TA_B200_ERR_UNSUPPORTED, "p must be in [0, 1], got %g", p->p);
    double total = 1.0;
    for (int d = 0; d < 4; ++d) {
        if (p->sizes[d] < 0) return fail(TA_B200_ERR_SHAPE, "size %d is negative", d);
        total *= (double)p->sizes[d];
    }
    if (total >= 4398046511104.0) return fail(TA_B200_ERR_TOO_LARGE, "at most 2^42 elements per call");
    if (total == 0.0) return TA_B200_OK;
    if (!p->x || !p->y) return fail(TA_B200_ERR_NULL, "x/y is NULL");
    if (((uintptr_t)p->x | (uintptr_t)p->y | (uintptr_t)p->residual) % es || (uintptr_t)p->seed_ptr % 8)
        return fail(TA_B200_ERR_UNSUPPORTED, "tensors must be aligned to their elements");
    DeviceState *s = nullptr;
    int rc = current_device(&s, nullptr);
    if (rc != TA_B200_OK) return rc;

    DropoutArgs a;
    memset(&a, 0, sizeof(a));
    a.x = p->x; a.residual = p->residual; a.y = p->y;
    a.seed = p->seed; a.seed_ptr = p->seed_ptr; a.offset = p->offset;
    a.numel = (long long)total;
    // Merge neighbouring dimensions that are shared or counted alike, innermost first: the fewer, the
    // fewer divisions in the kernel.  A dimension of size one merges with anything.
    int count = 0;
    long long size[4] = {1, 1, 1, 1};
    bool shared[4] = {false, false, false, false};
    for (int d = 3; d >= 0; --d) {
        if (p->sizes[d] == 1) continue;
        const bool sh = (p->shared >> d) & 1u;
        if (count > 0 && shared[count - 1] == sh) size[count - 1] *= p->sizes[d];
        else { size[count] = p->sizes[d]; shared[count] = sh; ++count; }
    }
    for (int d = 0; d < 4; ++d) { a.size[d] = 1; a.mstride[d] = 0; }
    long long stride = 1;
    for (int i = 0; i < count; ++i) {
        a.size[3 - i] = size[i];
        a.mstride[3 - i] = shared[i] ? 0 : stride;
        if (!shared[i]) stride *= size[i];
    }
    const double scaled = p->p * 4294967296.0;
    const uint64_t thr = (uint64_t)nearbyint(scaled);               // p = 1: 2^32, above every number
    a.drop_all = thr >> 32 != 0;
    a.thr_hi = (uint32_t)(thr >> 16) & 0xFFFFu;
    a.thr_lo = (uint32_t)(thr & 0xFFFFu);
    if (a.numel < (1LL << 32))
        for (int d = 0; d < 4; ++d) a.div[d] = fast_div_of((uint32_t)a.size[d]);
    a.scale = p->p < 1.0 ? (float)(1.0 / (1.0 - p->p)) : 0.0f;
    a.sm_count = s->sm_count;
    cudaError_t e = launch_dropout(a, p->dtype, stream);
    if (e != cudaSuccess) return cuda_fail(e, "launch(dropout)");
    return TA_B200_OK;
}

// ----------------------------------------------------------------------------- rotary positions
static int rotary(const ta_b200_rotary_params *p, cudaStream_t stream)
{
    if (!p) return fail(TA_B200_ERR_NULL, "params is NULL");
    if (p->struct_size != sizeof(ta_b200_rotary_params))
        return fail(TA_B200_ERR_SHAPE, "struct_size %u is not %zu (ABI mismatch)", p->struct_size, sizeof(ta_b200_rotary_params));
    const size_t es = feature_bytes(p->dtype);
    if (!es) return fail(TA_B200_ERR_DTYPE, "dtype %d", p->dtype);
    if (p->n < 0 || p->tokens < 0 || p->prefix < 0 || p->prefix > p->tokens || p->q_heads < 0 || p->k_heads < 0 || p->dim <= 0)
        return fail(TA_B200_ERR_SHAPE, "bad sizes n=%lld tokens=%lld prefix=%d heads=%d/%d dim=%d", (long long)p->n,
                    (long long)p->tokens, p->prefix, p->q_heads, p->k_heads, p->dim);
    if (p->axes < 1 || p->axes > 3) return fail(TA_B200_ERR_UNSUPPORTED, "one to three axes, got %d", p->axes);
    int rot = 0;
    for (int i = 0; i < p->axes; ++i) {
        if (p->sections[i] < 0 || p->sections[i] % 2) return fail(TA_B200_ERR_SHAPE, "sections must be even and not negative");
        if (p->sections[i] > p->dim) return fail(TA_B200_ERR_SHAPE, "sections add up to more than the head dimension %d", p->dim);
        rot += p->sections[i];
    }
    if (rot > p->dim) return fail(TA_B200_ERR_SHAPE, "sections add up to more than the head dimension %d", p->dim);
    if (rot / 2 > kRotaryMaxPairs) return fail(TA_B200_ERR_TOO_LARGE, "at most %d rotated elements per head", 2 * kRotaryMaxPairs);
    if (p->tokens >= (1LL << 31) || p->dim > 65536 || p->q_heads > 65536 || p->k_heads > 65536 || (double)p->n * p->tokens * p->dim >= 4398046511104.0)
        return fail(TA_B200_ERR_TOO_LARGE, "tokens below 2^31, head dimension and heads up to 65536, 2^42 elements per head");
    if (!(p->base > 0.0)) return fail(TA_B200_ERR_UNSUPPORTED, "base must be positive");
    if (p->pairing != TA_B200_PAIR_INTERLEAVED && p->pairing != TA_B200_PAIR_HALVES) return fail(TA_B200_ERR_UNSUPPORTED, "pairing %d", p->pairing);
    if (p->spectrum != TA_B200_SPECTRUM_AXIS && p->spectrum != TA_B200_SPECTRUM_JOINT)
        return fail(TA_B200_ERR_UNSUPPORTED, "spectrum %d", p->spectrum);
    if (p->position_kind < TA_B200_POS_GRID || p->position_kind > TA_B200_POS_I32)
        return fail(TA_B200_ERR_UNSUPPORTED, "position kind %d", p->position_kind);
    if (p->position_kind == TA_B200_POS_GRID) {
        double cells = 1.0;
        for (int i = 0; i < p->axes; ++i) {
            if (p->grid[i] < 0) return fail(TA_B200_ERR_SHAPE, "grid sizes must not be negative");
            cells *= p->grid[i];
        }
        if (cells != (double)(p->tokens - p->prefix))
            return fail(TA_B200_ERR_SHAPE, "the grid has %.0f cells for %lld tokens", cells, (long long)(p->tokens - p->prefix));
        if (!(p->patch > 0.0f)) return fail(TA_B200_ERR_UNSUPPORTED, "patch must be positive");
        if (p->top && p->axes < 2) return fail(TA_B200_ERR_UNSUPPORTED, "top needs a height axis");
    }
    if (p->n == 0 || p->tokens == 0 || p->q_heads + p->k_heads == 0) return TA_B200_OK;
    if ((p->q_heads > 0 && (!p->q || !p->q_out)) || (p->k_heads > 0 && (!p->k || !p->k_out)))
        return fail(TA_B200_ERR_NULL, "q/k or their outputs are NULL");
    if (p->position_kind != TA_B200_POS_GRID && !p->positions && p->tokens > p->prefix) return fail(TA_B200_ERR_NULL, "positions is NULL");
    if (((uintptr_t)p->q | (uintptr_t)p->k | (uintptr_t)p->q_out | (uintptr_t)p->k_out) % es ||
        (uintptr_t)p->positions % (p->position_kind == TA_B200_POS_I64 ? 8 : 4) || ((uintptr_t)p->top | (uintptr_t)p->left) % 4)
        return fail(TA_B200_ERR_UNSUPPORTED, "tensors must be aligned to their elements");
    DeviceState *s = nullptr;
    int rc = current_device(&s, nullptr);
    if (rc != TA_B200_OK) return rc;

    RotaryArgs a;
    memset(&a, 0, sizeof(a));
    a.q = p->q; a.k = p->k; a.q_out = p->q_out; a.k_out = p->k_out;
    for (int i = 0; i < 3; ++i) {
        a.qs[i] = p->q_strides[i]; a.ks[i] = p->k_strides[i];
        a.qos[i] = p->q_out_strides[i]; a.kos[i] = p->k_out_strides[i];
        a.pos_s[i] = p->position_strides[i];
        a.grid[i] = p->grid[i] > 0 ? p->grid[i] : 1;
    }
    for (int i = 0; i < 3; ++i) a.grid_div[i] = fast_div_of((uint32_t)a.grid[i]);
    a.token_div = fast_div_of((uint32_t)p->tokens);
    a.n = p->n; a.tokens = p->tokens; a.prefix = p->prefix; a.q_heads = p->q_heads; a.k_heads = p->k_heads; a.dim = p->dim;
    a.axes = p->axes; a.pairs = rot / 2; a.halves = p->pairing == TA_B200_PAIR_HALVES; a.inverse = p->inverse != 0;
    a.pos_kind = p->position_kind; a.positions = p->positions; a.patch = p->patch;
    a.top = p->top; a.left = p->left; a.flip = p->flip;
    a.sm_count = s->sm_count;
    const double log_base = log(p->base), per = p->position_kind == TA_B200_POS_GRID ? (double)p->patch : 1.0;
    int j = 0;
    for (int i = 0; i < 3; ++i) {
        const int half = i < p->axes ? p->sections[i] / 2 : 0;
        for (int m = 0; m < half; ++m, ++j) {
            const double power = p->spectrum == TA_B200_SPECTRUM_AXIS ? (double)m / half : 2.0 * j / rot;
            const double turns = exp(-power * log_base) / (6.283185307179586476925 * per);
            a.freq_hi[j] = (float)turns;
            a.freq_lo[j] = (float)(turns - (double)a.freq_hi[j]);
        }
        a.axis_end[i] = j;
    }
    cudaError_t e = launch_rotary(a, p->dtype, stream);
    if (e != cudaSuccess) return cuda_fail(e, "launch(rotary)");
    return TA_B200_OK;
}

}  // namespace ta

extern "C" {

int ta_b200_group_norm(const ta_b200_group_norm_params *p, void *stream) { return ta::group_norm(p, false, (cudaStream_t)stream); }
int ta_b200_group_norm_backward(const ta_b200_group_norm_params *p, void *stream) { return ta::group_norm(p, true, (cudaStream_t)stream); }

size_t ta_b200_group_norm_scratch_bytes(const ta_b200_group_norm_params *p, int32_t backward)
{
    ta::GnArgs a;
    if (ta::group_norm_args(p, backward != 0, a) != TA_B200_OK || a.n == 0 || a.rows == 0) return 0;
    ta::DeviceState *s = nullptr;
    if (ta::current_device(&s, nullptr) != TA_B200_OK) return 0;
    a.sm_count = s->sm_count;
    return ta::group_norm_scratch(p->dtype, a, backward != 0);
}

int ta_b200_dropout(const ta_b200_dropout_params *p, void *stream) { return ta::dropout(p, (cudaStream_t)stream); }
int ta_b200_rotary(const ta_b200_rotary_params *p, void *stream) { return ta::rotary(p, (cudaStream_t)stream); }

}  // extern "C"
