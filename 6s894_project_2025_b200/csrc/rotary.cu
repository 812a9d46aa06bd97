// Position rotation of queries and keys, alone or behind an RMS norm of every head, with the Hadamard rotation of the
// head dimension in the same pass, and the gradients of both.
//
// One row is one head of one token: D values, rounded to the tensor's type once, on the store.  With R = 2 * pairs
// rotated dimensions and angle_i = positions[axis(i)] * inv_freq[i],
//     forward   n = x * rsqrt(mean(x^2) + eps) * w        (norm only)
//               y = n with (a, b) -> (a cos - b sin, b cos + a sin) for every pair i: dimensions (i, i + pairs), or
//                   (2i, 2i + 1) when interleaved; dimensions from R on stay
//               y = y . H_D / sqrt(D)                      (hadamard only)
//     gradient  the transposed steps in reverse order: H is symmetric, the rotation's transpose is the rotation by
//               -angle, and for the norm with h = x * r, r = rsqrt(mean(x^2) + eps)
//                   dw = sum over rows of g * h,     dx = r * (g * w - h * mean(g * w * h)).
// Everything between the load and the store is fp32; the angle is reduced in fp64 (a position of 10^6 times a frequency
// has no correct digits left in fp32 once it is taken modulo 2 pi).
//
// There is no counterpart in the reference, whose only operation on heads is the plain transform along the last
// dimension (csrc/hadamard_transform.cpp:12-70).
#include "common.cuh"

namespace b200ht {

constexpr int kMaxHeadDim = 256;
constexpr int kMaxAxes = 4;

struct RotTensor {
    const void *x;      // input rows
    const void *g;      // gradient of the output rows (gradient kernels only)
    void *y;            // output rows
    const void *w;      // norm weight, D values
    long long x_tok, x_head, g_tok, g_head, y_tok, y_head;   // strides in elements
    int heads;
};

struct RotArgs {
    RotTensor t[2];     // queries, keys
    const void *pos;
    long long pos_axis, pos_tok;   // strides in elements
    const float *inv_freq;
    float *partial;     // gradient of the weights: one row of D floats per block
    int tokens, D, pairs;
    int pos64, w_f32, interleaved, inverse;
    float eps;
    unsigned char axis[kMaxHeadDim / 2];
};

// cos and sin of position * frequency.  The angle in turns is reduced to [-1/2, 1/2] in fp64, where the product of a
// 32-bit position and a frequency is good to 2^-21 turns at worst; the rest is good to a few 2^-24.
__device__ __forceinline__ float2 rot_cos_sin(const RotArgs &a, int token, int pair)
{
    const long long at = (long long)a.axis[pair] * a.pos_axis + (long long)token * a.pos_tok;
    const double p = a.pos64 ? (double)((const long long *)a.pos)[at] : (double)((const int *)a.pos)[at];
    double u = p * ((double)a.inv_freq[pair] * 0.15915494309189533577);
    u -= rint(u);
    float s, c;
    sincospif(2.f * (float)u, &s, &c);
    return make_float2(c, s);
}

template <int DT>
__device__ __forceinline__ float rot_load(const void *p, long long i)
{
    if constexpr (DT == B200HT_F32) return ((const float *)p)[i];
    else if constexpr (DT == B200HT_BF16) return __bfloat162float(((const __nv_bfloat16 *)p)[i]);
    else return __half2float(((const __half *)p)[i]);
}
template <int DT>
__device__ __forceinline__ void rot_store(void *p, long long i, float v)
{
    if constexpr (DT == B200HT_F32) ((float *)p)[i] = v;
    else if constexpr (DT == B200HT_BF16) ((__nv_bfloat16 *)p)[i] = __float2bfloat16_rn(v);
    else ((__half *)p)[i] = __float2half_rn(v);
}
template <int DT>
__device__ __forceinline__ float rot_weight(const RotArgs &a, const void *w, int i)
{
    return a.w_f32 ? ((const float *)w)[i] : rot_load<DT>(w, i);
}

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// ---------------------------------------------------------------------------
// Any head dimension, stride and alignment: a warp per row, the row in shared memory as fp32, one element per lane and
// step.
// ---------------------------------------------------------------------------
constexpr int kAnyWarps = 4;

// y = y . H_D / sqrt(D) on a row in shared memory, by one warp.
__device__ __forceinline__ void any_hadamard(float *row, int D, int lane)
{
    for (int h = 1; h < D; h <<= 1) {
        for (int i = lane; i < D / 2; i += 32) {
            const int lo = ((i & ~(h - 1)) << 1) | (i & (h - 1));
            const float u = row[lo], v = row[lo + h];
            row[lo] = u + v;
            row[lo + h] = u - v;
        }
        __syncwarp();
    }
    const float c = rsqrtf((float)D);
    for (int i = lane; i < D; i += 32) row[i] *= c;
    __syncwarp();
}

__device__ __forceinline__ void any_rotate(const RotArgs &a, float *row, int token, float sign, int lane)
{
    for (int i = lane; i < a.pairs; i += 32) {
        const float2 cs = rot_cos_sin(a, token, i);
        const int lo = a.interleaved ? 2 * i : i, hi = a.interleaved ? 2 * i + 1 : i + a.pairs;
        const float u = row[lo], v = row[hi], s = sign * cs.y;
        row[lo] = u * cs.x - v * s;
        row[hi] = v * cs.x + u * s;
    }
    __syncwarp();
}

template <int DT, bool NORM, bool HAD>
__global__ void __launch_bounds__(32 * kAnyWarps) rotary_any_kernel(const __grid_constant__ RotArgs a)
{
    __shared__ float rows[kAnyWarps][kMaxHeadDim];
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int heads = a.t[0].heads + a.t[1].heads;
    const long long n = (long long)a.tokens * heads;
    float *row = rows[warp];
    for (long long r = (long long)blockIdx.x * kAnyWarps + warp; r < n; r += (long long)gridDim.x * kAnyWarps) {
        const int token = (int)(r / heads);
        int h = (int)(r - (long long)token * heads);
        const int which = h < a.t[0].heads ? 0 : 1;
        if (which) h -= a.t[0].heads;
        const RotTensor &t = a.t[which];
        const long long xo = token * t.x_tok + h * t.x_head, yo = token * t.y_tok + h * t.y_head;
        float sum = 0.f;
        for (int i = lane; i < a.D; i += 32) {
            const float v = rot_load<DT>(t.x, xo + i);
            row[i] = v;
            sum = fmaf(v, v, sum);
        }
        __syncwarp();
        if constexpr (NORM) {
            const float rs = rsqrtf(warp_sum(sum) / (float)a.D + a.eps);
            for (int i = lane; i < a.D; i += 32) row[i] = row[i] * rs * rot_weight<DT>(a, t.w, i);
            __syncwarp();
        }
        if (HAD && a.inverse) any_hadamard(row, a.D, lane);
        any_rotate(a, row, token, a.inverse ? -1.f : 1.f, lane);
        if (HAD && !a.inverse) any_hadamard(row, a.D, lane);
        for (int i = lane; i < a.D; i += 32) rot_store<DT>(t.y, yo + i, row[i]);
        __syncwarp();
    }
}

// Gradient of the norm and rotation.  The blocks from `first` on (`blocks` of them) serve this tensor; each warp sums
// g * h over its rows, the warps of a block are added in order, and the block's row of `partial` goes to the second
// kernel, so the result does not depend on timing.
template <int DT, bool HAD>
__global__ void __launch_bounds__(32 * kAnyWarps)
norm_rotary_any_grad_kernel(const __grid_constant__ RotArgs a, int q_blocks)
{
    __shared__ float rows[kAnyWarps][kMaxHeadDim];
    __shared__ float sums[kAnyWarps][kMaxHeadDim];
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int which = (int)blockIdx.x < q_blocks ? 0 : 1;
    const int block = which ? (int)blockIdx.x - q_blocks : (int)blockIdx.x;
    const int blocks = which ? (int)gridDim.x - q_blocks : q_blocks;
    const RotTensor &t = a.t[which];
    const long long n = (long long)a.tokens * t.heads;
    float *row = rows[warp];
    for (int i = lane; i < a.D; i += 32) sums[warp][i] = 0.f;
    for (long long r = (long long)block * kAnyWarps + warp; r < n; r += (long long)blocks * kAnyWarps) {
        const int token = (int)(r / t.heads), h = (int)(r - (long long)token * t.heads);
        const long long xo = token * t.x_tok + h * t.x_head, go = token * t.g_tok + h * t.g_head;
        const long long yo = token * t.y_tok + h * t.y_head;
        float sum = 0.f;
        for (int i = lane; i < a.D; i += 32) {
            const float v = rot_load<DT>(t.x, xo + i);
            sum = fmaf(v, v, sum);
            row[i] = rot_load<DT>(t.g, go + i);
        }
        __syncwarp();
        const float rs = rsqrtf(warp_sum(sum) / (float)a.D + a.eps);
        if (HAD) any_hadamard(row, a.D, lane);
        any_rotate(a, row, token, -1.f, lane);
        float dot = 0.f;
        for (int i = lane; i < a.D; i += 32) {
            const float hx = rot_load<DT>(t.x, xo + i) * rs;
            sums[warp][i] = fmaf(row[i], hx, sums[warp][i]);
            dot = fmaf(row[i] * rot_weight<DT>(a, t.w, i), hx, dot);
        }
        dot = warp_sum(dot) / (float)a.D;
        for (int i = lane; i < a.D; i += 32) {
            const float hx = rot_load<DT>(t.x, xo + i) * rs;
            rot_store<DT>(t.y, yo + i, rs * (row[i] * rot_weight<DT>(a, t.w, i) - hx * dot));
        }
        __syncwarp();
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.D; i += blockDim.x) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < kAnyWarps; ++w) s += sums[w][i];
        a.partial[(long long)blockIdx.x * a.D + i] = s;
    }
}

// dw[i] = sum of the blocks' rows, in a fixed order: 8 warps take every eighth row of 32 columns, then the warps are
// added in order.  blockIdx.y: queries or keys.
template <int DT>
__global__ void __launch_bounds__(256)
norm_weight_grad_kernel(const float *partial, int q_blocks, int k_blocks, int D, void *dwq, void *dwk, int w_f32)
{
    __shared__ float part[8][32];
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int i = blockIdx.x * 32 + lane;
    const float *rows = partial + (blockIdx.y ? (long long)q_blocks * D : 0);
    const int n = blockIdx.y ? k_blocks : q_blocks;
    float s = 0.f;
    if (i < D)
        for (int r = warp; r < n; r += 8) s += rows[(long long)r * D + i];
    part[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && i < D) {
        s = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) s += part[w][lane];
        void *dw = blockIdx.y ? dwk : dwq;
        if (w_f32) ((float *)dw)[i] = s;
        else rot_store<DT>(dw, i, s);
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
template <int DT, bool NORM>
static int launch_any(const RotArgs &a, bool had, cudaStream_t st)
{
    const long long rows = (long long)a.tokens * (a.t[0].heads + a.t[1].heads);
    const long long want = (rows + kAnyWarps - 1) / kAnyWarps, cap = (long long)sm_count() * 16;
    const dim3 grid((unsigned)(want < cap ? want : cap)), block(32 * kAnyWarps);
    return had ? launch_pdl(rotary_any_kernel<DT, NORM, true>, grid, block, 0, st, a)
               : launch_pdl(rotary_any_kernel<DT, NORM, false>, grid, block, 0, st, a);
}

// Blocks of the gradient kernel that serve the queries and the keys: shares of the rows, at least one each where there
// are rows.  `most` bounds the sum (the size of the workspace goes by it).
struct GradBlocks {
    int q, k;
};
static GradBlocks grad_blocks(long long q_rows, long long k_rows, long long rows_per_block, int most)
{
    const long long want = (q_rows + k_rows + rows_per_block - 1) / rows_per_block;
    const long long n = want < most ? want : most;
    GradBlocks b{0, 0};
    if (q_rows + k_rows == 0) return b;
    b.q = q_rows ? (int)(n * q_rows / (q_rows + k_rows)) : 0;
    if (q_rows && b.q < 1) b.q = 1;
    b.k = k_rows ? (int)(n - b.q) : 0;
    if (k_rows && b.k < 1) b.k = 1;
    return b;
}
constexpr int kGradBlocks = 148 * 8;   // blocks of a gradient launch at most (one more may come from rounding up)

static int check_rot_common(const RotArgs &a, int dtype, int flags, const unsigned char *axis_of_pair, int n_axes)
{
    if (dtype != B200HT_F16 && dtype != B200HT_BF16 && dtype != B200HT_F32) return B200HT_ERR_DTYPE;
    if (flags & ~(B200HT_ROT_INTERLEAVED | B200HT_ROT_HADAMARD | B200HT_ROT_INVERSE | B200HT_ROT_POS64 | B200HT_ROT_WEIGHT_F32))
        return B200HT_ERR_SIZE;
    if (a.tokens < 0 || a.t[0].heads < 0 || a.t[1].heads < 0) return B200HT_ERR_SIZE;
    if (a.D < 2 || a.D > kMaxHeadDim || (a.D & 1) || a.pairs < 1 || 2 * a.pairs > a.D) return B200HT_ERR_SIZE;
    if ((flags & B200HT_ROT_HADAMARD) && !is_pow2((uint64_t)a.D)) return B200HT_ERR_SIZE;
    if (n_axes < 1 || n_axes > kMaxAxes || (n_axes > 1 && !axis_of_pair)) return B200HT_ERR_SIZE;
    if (axis_of_pair)
        for (int i = 0; i < a.pairs; ++i)
            if (axis_of_pair[i] >= n_axes) return B200HT_ERR_SIZE;
    return 0;
}
static void fill_rot_common(RotArgs &a, int flags, const unsigned char *axis_of_pair)
{
    a.interleaved = (flags & B200HT_ROT_INTERLEAVED) ? 1 : 0;
    a.inverse = (flags & B200HT_ROT_INVERSE) ? 1 : 0;
    a.pos64 = (flags & B200HT_ROT_POS64) ? 1 : 0;
    a.w_f32 = (flags & B200HT_ROT_WEIGHT_F32) ? 1 : 0;
    for (int i = 0; i < kMaxHeadDim / 2; ++i) a.axis[i] = (axis_of_pair && i < a.pairs) ? axis_of_pair[i] : 0;
}
static bool misaligned(const void *p, int dtype) { return ((uintptr_t)p & (dtype == B200HT_F32 ? 3u : 1u)) != 0; }
static int check_rot_pointers(const RotArgs &a, int dtype, int flags)
{
    if (!a.pos || !a.inv_freq) return B200HT_ERR_NULL;
    if (((uintptr_t)a.pos & ((flags & B200HT_ROT_POS64) ? 7u : 3u)) || ((uintptr_t)a.inv_freq & 3u)) return B200HT_ERR_ALIGN;
    for (int i = 0; i < 2; ++i) {
        if (!a.t[i].heads) continue;
        if (!a.t[i].x || !a.t[i].y) return B200HT_ERR_NULL;
        if (misaligned(a.t[i].x, dtype) || misaligned(a.t[i].y, dtype) || misaligned(a.t[i].g, dtype)) return B200HT_ERR_ALIGN;
        if (misaligned(a.t[i].w, (flags & B200HT_ROT_WEIGHT_F32) ? B200HT_F32 : dtype)) return B200HT_ERR_ALIGN;
    }
    return 0;
}

template <int DT>
static int launch_rotary(const RotArgs &a, bool norm, bool had, cudaStream_t st)
{
    return norm ? launch_any<DT, true>(a, had, st) : launch_any<DT, false>(a, had, st);
}

template <int DT>
static int launch_norm_grad(const RotArgs &a, bool had, void *dwq, void *dwk, cudaStream_t st)
{
    const long long q_rows = (long long)a.tokens * a.t[0].heads, k_rows = (long long)a.tokens * a.t[1].heads;
    const GradBlocks b = grad_blocks(q_rows, k_rows, kAnyWarps, kGradBlocks);
    if (b.q + b.k) {
        const dim3 grid((unsigned)(b.q + b.k)), block(32 * kAnyWarps);
        const int rc = had ? launch_pdl(norm_rotary_any_grad_kernel<DT, true>, grid, block, 0, st, a, b.q)
                           : launch_pdl(norm_rotary_any_grad_kernel<DT, false>, grid, block, 0, st, a, b.q);
        if (rc) return rc;
    }
    return launch_pdl(norm_weight_grad_kernel<DT>, dim3((unsigned)((a.D + 31) / 32), 2), dim3(256), 0, st, (const float *)a.partial,
                      b.q, b.k, a.D, dwq, dwk, a.w_f32);
}

}  // namespace b200ht

extern "C" int b200ht_rotary_qk(const void *q, const void *k, void *q_out, void *k_out, const void *q_weight,
                                const void *k_weight, float eps, int tokens, int q_heads, int k_heads, int head_dim,
                                const long long *strides, int dtype, const void *positions, long long pos_axis_stride,
                                long long pos_token_stride, int n_axes, const unsigned char *axis_of_pair,
                                const float *inv_freq, int pairs, int flags, void *stream)
{
    using namespace b200ht;
    RotArgs a{};
    a.tokens = tokens;
    a.D = head_dim;
    a.pairs = pairs;
    a.t[0].heads = q_heads;
    a.t[1].heads = k_heads;
    int rc = check_rot_common(a, dtype, flags, axis_of_pair, n_axes);
    if (rc) return rc;
    const bool norm = q_weight || k_weight;
    if (norm && (flags & B200HT_ROT_INVERSE)) return B200HT_ERR_SIZE;   // the norm's gradient is b200ht_norm_rotary_qk_backward
    if (tokens == 0 || q_heads + k_heads == 0) return 0;
    if (!strides || (norm && ((q_heads && !q_weight) || (k_heads && !k_weight)))) return B200HT_ERR_NULL;
    a.t[0].x = q; a.t[0].y = q_out; a.t[0].w = q_weight;
    a.t[1].x = k; a.t[1].y = k_out; a.t[1].w = k_weight;
    a.t[0].x_tok = strides[0]; a.t[0].x_head = strides[1]; a.t[1].x_tok = strides[2]; a.t[1].x_head = strides[3];
    a.t[0].y_tok = strides[4]; a.t[0].y_head = strides[5]; a.t[1].y_tok = strides[6]; a.t[1].y_head = strides[7];
    a.pos = positions;
    a.pos_axis = pos_axis_stride;
    a.pos_tok = pos_token_stride;
    a.inv_freq = inv_freq;
    a.eps = eps;
    fill_rot_common(a, flags, axis_of_pair);
    rc = check_rot_pointers(a, dtype, flags);
    if (rc) return rc;
    rc = check_device();
    if (rc) return rc;
    const bool had = (flags & B200HT_ROT_HADAMARD) != 0;
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == B200HT_F32) return launch_rotary<B200HT_F32>(a, norm, had, st);
    if (dtype == B200HT_BF16) return launch_rotary<B200HT_BF16>(a, norm, had, st);
    return launch_rotary<B200HT_F16>(a, norm, had, st);
}

extern "C" size_t b200ht_norm_rotary_qk_backward_workspace_bytes(int head_dim)
{
    if (head_dim < 2 || head_dim > b200ht::kMaxHeadDim) return 0;
    return (size_t)(b200ht::kGradBlocks + 1) * (size_t)head_dim * sizeof(float);
}

extern "C" int b200ht_norm_rotary_qk_backward(const void *dq_out, const void *dk_out, const void *q, const void *k,
                                              const void *q_weight, const void *k_weight, float eps, void *dq, void *dk,
                                              void *dq_weight, void *dk_weight, int tokens, int q_heads, int k_heads,
                                              int head_dim, const long long *strides, int dtype, const void *positions,
                                              long long pos_axis_stride, long long pos_token_stride, int n_axes,
                                              const unsigned char *axis_of_pair, const float *inv_freq, int pairs,
                                              int flags, void *workspace, size_t workspace_bytes, void *stream)
{
    using namespace b200ht;
    RotArgs a{};
    a.tokens = tokens;
    a.D = head_dim;
    a.pairs = pairs;
    a.t[0].heads = q_heads;
    a.t[1].heads = k_heads;
    int rc = check_rot_common(a, dtype, flags, axis_of_pair, n_axes);
    if (rc) return rc;
    if (flags & B200HT_ROT_INVERSE) return B200HT_ERR_SIZE;
    if (!strides || !q_weight || !k_weight || !dq_weight || !dk_weight) return B200HT_ERR_NULL;
    if (!workspace || workspace_bytes < b200ht_norm_rotary_qk_backward_workspace_bytes(head_dim)) return B200HT_ERR_WORKSPACE;
    if (!aligned16(workspace)) return B200HT_ERR_ALIGN;
    const int wdt = (flags & B200HT_ROT_WEIGHT_F32) ? B200HT_F32 : dtype;
    if (misaligned(dq_weight, wdt) || misaligned(dk_weight, wdt) || misaligned(q_weight, wdt) || misaligned(k_weight, wdt))
        return B200HT_ERR_ALIGN;
    a.t[0].x = q; a.t[0].g = dq_out; a.t[0].y = dq; a.t[0].w = q_weight;
    a.t[1].x = k; a.t[1].g = dk_out; a.t[1].y = dk; a.t[1].w = k_weight;
    for (int i = 0; i < 2; ++i) {
        a.t[i].g_tok = strides[2 * i]; a.t[i].g_head = strides[2 * i + 1];
        a.t[i].x_tok = strides[4 + 2 * i]; a.t[i].x_head = strides[5 + 2 * i];
        a.t[i].y_tok = strides[8 + 2 * i]; a.t[i].y_head = strides[9 + 2 * i];
    }
    a.pos = positions;
    a.pos_axis = pos_axis_stride;
    a.pos_tok = pos_token_stride;
    a.inv_freq = inv_freq;
    a.eps = eps;
    a.partial = (float *)workspace;
    fill_rot_common(a, flags, axis_of_pair);
    if (tokens > 0) {
        rc = check_rot_pointers(a, dtype, flags);
        if (rc) return rc;
        if ((q_heads && !dq_out) || (k_heads && !dk_out)) return B200HT_ERR_NULL;
    }
    rc = check_device();
    if (rc) return rc;
    const bool had = (flags & B200HT_ROT_HADAMARD) != 0;
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == B200HT_F32) return launch_norm_grad<B200HT_F32>(a, had, dq_weight, dk_weight, st);
    if (dtype == B200HT_BF16) return launch_norm_grad<B200HT_BF16>(a, had, dq_weight, dk_weight, st);
    return launch_norm_grad<B200HT_F16>(a, had, dq_weight, dk_weight, st);
}
