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
    int n_axes, pos64, w_f32, interleaved, inverse;
    float eps;
    unsigned char axis[kMaxHeadDim / 2];
};

// cos and sin of position * frequency.  The angle in turns is reduced to [-1/2, 1/2] in fp64, where the product of a
// 32-bit position and a frequency is good to 2^-21 turns at worst; the rest is good to a few 2^-24.
__device__ __forceinline__ float2 rot_cos_sin(const RotArgs &a, int token, int pair)
{
    const long long at = (a.n_axes > 1 ? a.axis[pair] * a.pos_axis : 0) + token * a.pos_tok;
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
// Any head dimension, stride, alignment and number of pairs: a warp per row, the row in shared memory as fp32, one element
// per lane and step.  Six to eleven times the floor (the fast form below 1.1 to 1.7), for rows that it does not take: heads
// that are no multiple of 16 (72: 311 us for 16384 x 40, floor 29), rows off a 16-byte boundary, and split pairs of which
// some dimensions stay where they are, unless they are a multiple of 8 in the first half of the head (128 with 96 turning:
// 320 us, with neighbouring pairs 58, floor 51; 80 with 40 turning: 201 us, floor 32).
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

// ---------------------------------------------------------------------------
// The fast form, for rows of 16-byte vectors: head_dim a multiple of 16, every row on a 16-byte boundary, and pairs that
// are neighbours, or halves of the whole head, or lie in its first half eight by eight.
//
// A group of LANES lanes (the power of two from head_dim / 16 on) holds a row in registers: lane j has dimensions
// 8j .. 8j + 7 and head_dim / 2 + the same, so both members of a split pair, and the top bit of the index for H, meet in
// one lane; H needs shuffles for log2(head_dim) - 4 bits only.  A block of 256 threads takes `tb` tokens: cos and sin of
// their pairs are computed once into shared memory and serve all heads, each group walks over heads of one token with
// the next row's loads in flight.  Bound: HBM without H, the instruction rate with it (160 issued instructions per 512
// values and warp, 330 with H), hence the packed fp32 instructions: 66 us against 73 without them.
// 16384 tokens x 40 heads x 128, bf16 (51 us at the copy bandwidth): rotation 59 us, with H 63, norm 64, norm with H 77; four
// resident blocks an SM (64 registers) measured best (62 / 66 / 65 / 76 then), three 65 / 70 / 68 / 77, five spill (68 / 104
// / 92 / 122).  fp32, 8192 x 18 x 256 (46 us): rotation 60 us, norm 63; a lane's 32 bytes leave as two halves of a sector.
// ---------------------------------------------------------------------------
constexpr int kRowThreads = 256;

__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;\n"
        : "=l"(reinterpret_cast<unsigned long long &>(d))
        : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;\n"
        : "=l"(reinterpret_cast<unsigned long long &>(d))
        : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)));
    return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n"
        : "=l"(reinterpret_cast<unsigned long long &>(d))
        : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)),
          "l"(reinterpret_cast<unsigned long long &>(c)));
    return d;
}
__device__ __forceinline__ float2 sub2(float2 a, float2 b)
{
    float2 d;
    asm("sub.rn.f32x2 %0, %1, %2;\n"
        : "=l"(reinterpret_cast<unsigned long long &>(d))
        : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)));
    return d;
}

// The two vectors of a lane as they lie in memory, and as fp32: v[s][i] = dimensions 2i, 2i + 1 of vector s.
template <int DT>
struct RowRaw {
    uint4 v[2][DT == B200HT_F32 ? 2 : 1];
};
// `p` is the lane's first vector; the second lies `half` bytes on.
template <int DT>
__device__ __forceinline__ void row_load(RowRaw<DT> &r, const unsigned char *p, int half)
{
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < (DT == B200HT_F32 ? 2 : 1); ++i) r.v[s][i] = ((const uint4 *)(p + s * half))[i];
}
template <int DT>
__device__ __forceinline__ void row_unpack(const RowRaw<DT> &r, float2 (&v)[2][4])
{
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        if constexpr (DT == B200HT_F32) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                v[s][2 * i] = make_float2(__uint_as_float(r.v[s][i].x), __uint_as_float(r.v[s][i].y));
                v[s][2 * i + 1] = make_float2(__uint_as_float(r.v[s][i].z), __uint_as_float(r.v[s][i].w));
            }
        } else {
            v[s][0] = unpack2<DT>(r.v[s][0].x);
            v[s][1] = unpack2<DT>(r.v[s][0].y);
            v[s][2] = unpack2<DT>(r.v[s][0].z);
            v[s][3] = unpack2<DT>(r.v[s][0].w);
        }
    }
}
template <int DT>
__device__ __forceinline__ void row_store(unsigned char *q, int half, const float2 (&v)[2][4])
{
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        uint4 *p = (uint4 *)(q + s * half);
        if constexpr (DT == B200HT_F32) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                p[i] = make_uint4(__float_as_uint(v[s][2 * i].x), __float_as_uint(v[s][2 * i].y),
                                  __float_as_uint(v[s][2 * i + 1].x), __float_as_uint(v[s][2 * i + 1].y));
        } else {
            p[0] = make_uint4(pack2<DT>(v[s][0].x, v[s][0].y), pack2<DT>(v[s][1].x, v[s][1].y),
                              pack2<DT>(v[s][2].x, v[s][2].y), pack2<DT>(v[s][3].x, v[s][3].y));
        }
    }
}
// Weights as the lanes read them: four dimensions (16 bytes) of each lane side by side.
template <int DT>
__device__ __forceinline__ void fill_weights(float *wts, const RotArgs &a, const void *w, int D, int lanes)
{
    for (int i = threadIdx.x; i < D; i += kRowThreads) {
        const int s = i / (D / 2), e = i - s * (D / 2);   // vector, dimension within the half
        wts[((2 * s + ((e >> 2) & 1)) * lanes + (e >> 3)) * 4 + (e & 3)] = rot_weight<DT>(a, w, i);
    }
}
__device__ __forceinline__ float4 row_weights(const float *wts, int s, int i, int j, int lanes)   // dimensions 4i .. 4i + 3
{
    return *(const float4 *)(wts + ((2 * s + i) * lanes + j) * 4);
}
template <int LANES>
__device__ __forceinline__ float row_sum(float v)
{
#pragma unroll
    for (int o = LANES / 2; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// y = y . H; `lanes` = D / 16 lanes hold the row.
template <int LANES>
__device__ __forceinline__ void row_hadamard(float2 (&v)[2][4], int j, int lanes)
{
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[s][i] = make_float2(v[s][i].x + v[s][i].y, v[s][i].x - v[s][i].y);
#pragma unroll
        for (int m = 1; m < 4; m <<= 1)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (!(i & m)) {
                    const float2 a = v[s][i], b = v[s][i | m];
                    v[s][i] = add2(a, b);
                    v[s][i | m] = sub2(a, b);
                }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 a = v[0][i], b = v[1][i];
        v[0][i] = add2(a, b);
        v[1][i] = sub2(a, b);
    }
#pragma unroll
    for (int m = 1; m < LANES; m <<= 1) {
        if (m < lanes) {
            const float sg = (j & m) ? -1.f : 1.f;
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 o = make_float2(__shfl_xor_sync(0xffffffffu, v[s][i].x, m),
                                                 __shfl_xor_sync(0xffffffffu, v[s][i].y, m));
                    v[s][i] = fma2(v[s][i], make_float2(sg, sg), o);
                }
        }
    }
}
__device__ __forceinline__ void row_scale(float2 (&v)[2][4], float c)
{
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[s][i] = mul2(v[s][i], make_float2(c, c));
}

// How the pairs lie in a lane's registers.
enum { kPairsNeighbour, kPairsHalves, kPairsInFirstHalf };

// cos and sin of the lane's pairs: c[i], s[i] are those of dimensions 2i, 2i + 1 of vector 0 (and of vector 1: split over
// the whole head, both vectors have the same pairs); for neighbours c[0..1] are vector 0's four pairs, c[2..3] vector 1's.
struct RowTurn {
    float2 c[4], s[4];
};

__device__ __forceinline__ void row_turn(RowTurn &t, const float2 *tab, int mode, int j, int D, int pairs)
{
    if (mode == kPairsNeighbour) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 cs = tab[(i >> 2) * (D / 4) + 4 * j + (i & 3)];
            (i & 1 ? t.c[i >> 1].y : t.c[i >> 1].x) = cs.x;
            (i & 1 ? t.s[i >> 1].y : t.s[i >> 1].x) = cs.y;
        }
        return;
    }
    // split pairs in the first half: the second member's lane has them `pairs` dimensions on, with sin's sign turned
    const int e = 8 * j;
    const bool second = mode == kPairsInFirstHalf && e >= pairs;
    const bool none = mode == kPairsInFirstHalf && e >= 2 * pairs;
    const int first = second ? e - pairs : e;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float2 cs = none ? make_float2(1.f, 0.f) : tab[first + i];
        (i & 1 ? t.c[i >> 1].y : t.c[i >> 1].x) = cs.x;
        (i & 1 ? t.s[i >> 1].y : t.s[i >> 1].x) = mode == kPairsInFirstHalf && !second ? -cs.y : cs.y;
    }
}

// Dimensions behind the pairs are not touched: times 1 and 0, an infinity among them would be NaN and reach its neighbour.
__device__ __forceinline__ void row_rotate(float2 (&v)[2][4], const RowTurn &t, int mode, int partner, int j, int D, int pairs)
{
    if (mode == kPairsHalves) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 a = v[0][i], b = v[1][i];
            v[0][i] = sub2(mul2(a, t.c[i]), mul2(b, t.s[i]));
            v[1][i] = fma2(b, t.c[i], mul2(a, t.s[i]));
        }
    } else if (mode == kPairsNeighbour) {
        const auto turn = [&](int s, int i) {
            const float c = i & 1 ? t.c[2 * s + (i >> 1)].y : t.c[2 * s + (i >> 1)].x;
            const float sn = i & 1 ? t.s[2 * s + (i >> 1)].y : t.s[2 * s + (i >> 1)].x;
            const float a = v[s][i].x, b = v[s][i].y;
            v[s][i] = make_float2(a * c - b * sn, b * c + a * sn);
        };
        if (2 * pairs == D) {
#pragma unroll
            for (int i = 0; i < 8; ++i) turn(i >> 2, i & 3);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if ((i >> 2) * (D / 4) + 4 * j + (i & 3) < pairs) turn(i >> 2, i & 3);
        }
    } else {
        const bool turns = partner != (int)(threadIdx.x & 31);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 o = make_float2(__shfl_sync(0xffffffffu, v[0][i].x, partner), __shfl_sync(0xffffffffu, v[0][i].y, partner));
            if (turns) v[0][i] = fma2(o, t.s[i], mul2(v[0][i], t.c[i]));
        }
    }
}

// cos and sin of `tb` tokens' pairs, D / 2 entries a token; entries behind the pairs turn nothing
// (SPLIT: a token's D / 2 cosines, then its sines).  By THREADS threads, a block or a warp.
template <int THREADS, bool SPLIT = false>
__device__ __forceinline__ void fill_turns(float2 *tab, const RotArgs &a, long long token0, int tb)
{
    const int half = a.D / 2;
    auto entry = [&](int tk, int pair) {
        float2 cs = make_float2(1.f, 0.f);
        if (pair < a.pairs && token0 + tk < a.tokens) {
            cs = rot_cos_sin(a, (int)token0 + tk, pair);
            if (a.inverse) cs.y = -cs.y;
        }
        if (SPLIT) {
            float *at = (float *)(tab + tk * half) + pair;
            at[0] = cs.x;
            at[half] = cs.y;
        } else {
            tab[tk * half + pair] = cs;
        }
    };
    if (THREADS == 32) {
        for (int tk = 0; tk < tb; ++tk)
            for (int pair = threadIdx.x % 32; pair < half; pair += 32) entry(tk, pair);
    } else {
        for (int i = threadIdx.x % THREADS; i < tb * half; i += THREADS) entry(i / half, i % half);
    }
}

// Lane of a warp that holds the other member of this lane's split pairs in the first half (pairs a multiple of 8).
__device__ __forceinline__ int row_partner(int mode, int j, int pairs)
{
    const int lane = threadIdx.x & 31;
    if (mode != kPairsInFirstHalf || 8 * j >= 2 * pairs) return lane;
    return 8 * j < pairs ? lane + pairs / 8 : lane - pairs / 8;
}

template <int DT, bool NORM, bool HAD, int LANES>
__global__ void __launch_bounds__(kRowThreads, DT == B200HT_F32 ? 2 : 4)
rotary_row_kernel(const __grid_constant__ RotArgs a, int tb, int mode)
{
    extern __shared__ float2 tab[];                  // [tb][D / 2], then the weights: [2][D] floats
    constexpr int GROUPS = kRowThreads / LANES, SIZE = DT == B200HT_F32 ? 4 : 2;
    const int D = a.D, half = D / 2, lanes = D / 16;
    float *wts = (float *)(tab + tb * half);
    const int group = threadIdx.x / LANES, j = threadIdx.x % LANES;
    const int per = GROUPS / tb, tk = group / per;   // groups of one token
    const int token0 = blockIdx.x * tb, token = token0 + tk;
    // the queries' heads come first, then the keys': each group has every per-th head
    const int q_steps = (a.t[0].heads + per - 1) / per, steps = q_steps + (a.t[1].heads + per - 1) / per;
    const bool mine = token < a.tokens && j < lanes;
    const int h0 = group - tk * per;
    pdl_launch_dependents();
    pdl_wait();

    const unsigned char *in;
    unsigned char *out;
    long long in_step, out_step;
    int left;                                        // heads of this tensor from the current one on
    auto start = [&](const RotTensor &t) {
        in = (const unsigned char *)t.x + (token * t.x_tok + h0 * t.x_head + 8 * j) * SIZE;
        in_step = per * t.x_head * SIZE;
        left = mine ? t.heads - h0 : 0;
    };
    auto start_out = [&](const RotTensor &t) {
        out = (unsigned char *)t.y + (token * t.y_tok + h0 * t.y_head + 8 * j) * SIZE;
        out_step = per * t.y_head * SIZE;
    };
    RowRaw<DT> next = {};
    start(q_steps ? a.t[0] : a.t[1]);
    start_out(q_steps ? a.t[0] : a.t[1]);
    if (left > 0) row_load<DT>(next, in, half * SIZE);
    fill_turns<kRowThreads>(tab, a, token0, tb);
    if constexpr (NORM) {
        if (a.t[0].heads) fill_weights<DT>(wts, a, a.t[0].w, D, lanes);
        if (a.t[1].heads) fill_weights<DT>(wts + D, a, a.t[1].w, D, lanes);
    }
    __syncthreads();
    RowTurn turn;
    const int jj = j < lanes ? j : 0;
    row_turn(turn, tab + tk * half, mode, jj, D, a.pairs);
    const int partner = row_partner(mode, j, a.pairs);
    const float hc = HAD ? rsqrtf((float)D) : 1.f, inv_d = 1.f / (float)D;

#pragma unroll 1
    for (int step = 0; step < steps; ++step) {
        const RowRaw<DT> cur = next;
        const bool on = left > 0;
        if (step + 1 == q_steps) {
            if (step + 1 < steps) start(a.t[1]);
        } else {
            in += in_step;
            left -= per;
        }
        if (step + 1 < steps && left > 0) row_load<DT>(next, in, half * SIZE);
        float2 v[2][4];
        row_unpack<DT>(cur, v);
        float scale = hc;                            // 1 / sqrt(D) of H and the norm's factor: linear, so once at the end
        if constexpr (NORM) {
            float2 q = make_float2(0.f, 0.f);
            const float *w = wts + (step < q_steps ? 0 : D);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float4 f = row_weights(w, s, i, jj, lanes);
                    q = fma2(v[s][2 * i], v[s][2 * i], q);
                    q = fma2(v[s][2 * i + 1], v[s][2 * i + 1], q);
                    v[s][2 * i] = mul2(v[s][2 * i], make_float2(f.x, f.y));
                    v[s][2 * i + 1] = mul2(v[s][2 * i + 1], make_float2(f.z, f.w));
                }
            const float sum = row_sum<LANES>(j < lanes ? q.x + q.y : 0.f);
            scale *= rsqrtf(sum * inv_d + a.eps);
        }
        if (HAD && !NORM && a.inverse) row_hadamard<LANES>(v, j, lanes);
        row_rotate(v, turn, mode, partner, jj, D, a.pairs);
        if (HAD && (NORM || !a.inverse)) row_hadamard<LANES>(v, j, lanes);
        if (HAD || NORM) row_scale(v, scale);
        if (on) row_store<DT>(out, half * SIZE, v);
        if (step + 1 == q_steps) {
            if (step + 1 < steps) start_out(a.t[1]);
        } else {
            out += out_step;
        }
    }
}

// Gradient of norm and rotation, the same layout of a row.  The first `q_blocks` blocks serve the queries, the others the
// keys.  A warp takes whole tokens (per = 32 / LANES / tokens-of-a-warp groups each) and needs no other warp until the
// end, where the block's share of the weights' gradient, in registers so far, is added up: with barriers around the
// table of cos and sin the blocks stood still for a fifth of the time.  Registers are what limits it: the next row comes
// by cp.async into a slot of shared memory that its own thread (fp32: group) alone reads, x is read from there once for
// each of its three uses, and for split pairs cos and sin stay in shared memory as well.  16384 tokens x 40 heads x 128,
// bf16: 90 - 95 us, 77 at the copy bandwidth; 127 with H (instruction rate).
__device__ __forceinline__ void copy_async16(uint32_t dst, const void *src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint4 load_shared16(uint32_t from)   // volatile: not kept in registers between two uses
{
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(from) : "memory");
    return v;
}
// Vector s of a row in its slot, as fp32.  `from`: 16 bits, the lane's first vector, the second 16 bytes a thread on; fp32,
// where the group's row begins, in its natural order, with `at` = byte of the lane's vector s.
template <int DT>
__device__ __forceinline__ void slot_vector(uint32_t from, int s, int at, float2 (&v)[4])
{
    if constexpr (DT == B200HT_F32) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint4 r = load_shared16(from + at + 16 * i);
            v[2 * i] = make_float2(__uint_as_float(r.x), __uint_as_float(r.y));
            v[2 * i + 1] = make_float2(__uint_as_float(r.z), __uint_as_float(r.w));
        }
    } else {
        const uint4 r = load_shared16(from + s * kRowThreads * 16);
        v[0] = unpack2<DT>(r.x);
        v[1] = unpack2<DT>(r.y);
        v[2] = unpack2<DT>(r.z);
        v[3] = unpack2<DT>(r.w);
    }
}
constexpr int kRowSlots = 2;   // 3 or 4 measured slower in 16 bits (108 us for 97 at 16384 x 40 x 128)
template <int DT>
constexpr int row_slot_bytes() { return kRowThreads * 16 * 4 * (DT == B200HT_F32 ? 2 : 1); }   // x and g, two vectors each

template <int DT, bool HAD, int LANES, int MODE>
__global__ void __launch_bounds__(kRowThreads, DT == B200HT_F32 ? 2 : 3)
norm_rotary_row_grad_kernel(const __grid_constant__ RotArgs a, int per_q, int per_k, int q_blocks)
{
    extern __shared__ __align__(16) unsigned char smem[];   // slots of rows, the warps' tables; at the end [groups][D] floats
    __shared__ __align__(16) float wts[kMaxHeadDim];
    constexpr int GROUPS = kRowThreads / LANES, SIZE = DT == B200HT_F32 ? 4 : 2, VECS = DT == B200HT_F32 ? 2 : 1;
    constexpr int SLOT = row_slot_bytes<DT>(), WARPS = kRowThreads / 32;
    const int D = a.D, half = D / 2, lanes = D / 16;
    const int which = (int)blockIdx.x < q_blocks ? 0 : 1;
    const RotTensor &t = a.t[which];
    const int per = which ? per_k : per_q;                  // groups of one token
    const int tokens = 32 / LANES / per;                    // tokens of a warp
    const int warp = threadIdx.x >> 5, group = threadIdx.x / LANES, j = threadIdx.x % LANES, jj = j < lanes ? j : 0;
    const int tk = group % (32 / LANES) / per, h0 = group % per;
    const int steps = (t.heads + per - 1) / per;
    const int partner = row_partner(MODE, j, a.pairs);
    const float hc = HAD ? rsqrtf((float)D) : 1.f, inv_d = 1.f / (float)D;
    // 16 bits: a lane copies the two vectors that it will read.  fp32: the lanes copy 16 bytes side by side, whole sectors
    // (their own 32 bytes would be two requests for half a sector each, and every sector would cross to the SM twice)
    const uint32_t slots = (uint32_t)__cvta_generic_to_shared(smem);
    const uint32_t copy_to = slots + (VECS == 2 ? group * LANES * 64 + j * 16 : threadIdx.x * 16);
    const uint32_t read_at = slots + (VECS == 2 ? group * LANES * 64 : threadIdx.x * 16);
    float2 *tab = (float2 *)(smem + kRowSlots * SLOT) + warp * tokens * half;
    pdl_launch_dependents();
    pdl_wait();
    fill_weights<DT>(wts, a, t.w, D, lanes);
    __syncthreads();

    float2 dw[2][4];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) dw[s][i] = make_float2(0.f, 0.f);

    // the rows on their way: kRowSlots - 1 steps ahead of the one at work
    const long long first = ((long long)(which ? (int)blockIdx.x - q_blocks : (int)blockIdx.x) * WARPS + warp) * tokens;
    const long long stride = (long long)(which ? (int)gridDim.x - q_blocks : q_blocks) * WARPS * tokens;
    const long long x_step = per * t.x_head * SIZE, g_step = per * t.g_head * SIZE, y_step = per * t.y_head * SIZE;
    const unsigned char *fx, *fg;
    long long f_first = first;
    int f_step = 0, f_left, slot = 0;
    auto row = [&]() {
        const long long token = f_first + tk;
        f_left = token < a.tokens && (VECS == 2 || j < lanes) ? t.heads - h0 : 0;
        fx = (const unsigned char *)t.x + (token * t.x_tok + h0 * t.x_head) * SIZE + 16 * j;
        fg = (const unsigned char *)t.g + (token * t.g_tok + h0 * t.g_head) * SIZE + 16 * j;
    };
    auto fetch = [&](int to_slot) {
        if (f_left > 0) {
            const uint32_t to = copy_to + to_slot * SLOT;
            if constexpr (VECS == 2) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (c * LANES + j < 4 * lanes) {
                        copy_async16(to + c * LANES * 16, fx + c * LANES * 16);
                        copy_async16(to + SLOT / 2 + c * LANES * 16, fg + c * LANES * 16);
                    }
            } else {
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    copy_async16(to + s * kRowThreads * 16, fx + s * half * SIZE);
                    copy_async16(to + SLOT / 2 + s * kRowThreads * 16, fg + s * half * SIZE);
                }
            }
        }
        asm volatile("cp.async.commit_group;\n" ::: "memory");
        if (++f_step == steps) {
            f_step = 0;
            f_first += stride;
            row();
        } else {
            fx += x_step;
            fg += g_step;
            f_left -= per;
        }
    };
    row();
#pragma unroll
    for (int i = 0; i + 1 < kRowSlots; ++i) fetch(i);
    for (long long token0 = first; token0 < a.tokens; token0 += stride) {
        __syncwarp();
        fill_turns<32, MODE == kPairsHalves>(tab, a, token0, tokens);   // a.inverse is set: the gradient turns back
        __syncwarp();
        RowTurn turn;
        if (MODE != kPairsHalves) row_turn(turn, tab + tk * half, MODE, jj, D, a.pairs);
        const uint32_t turns = (uint32_t)__cvta_generic_to_shared(tab + tk * half) + jj * 32;
        const long long token = token0 + tk;
        int left = token < a.tokens && j < lanes ? t.heads - h0 : 0;
        unsigned char *y = (unsigned char *)t.y + (token * t.y_tok + h0 * t.y_head + 8 * j) * SIZE;
#pragma unroll 1
        for (int step = 0; step < steps; ++step) {
            if (VECS == 2) __syncwarp();   // all lanes have read the slot that is filled now
            fetch(slot == 0 ? kRowSlots - 1 : slot - 1);
            asm volatile("cp.async.wait_group %0;\n" ::"n"(kRowSlots - 1) : "memory");
            if (VECS == 2) __syncwarp();   // and all have their copies here
            const bool on = left > 0;
            const uint32_t from_x = read_at + slot * SLOT, from_g = from_x + SLOT / 2;
            slot = slot + 1 == kRowSlots ? 0 : slot + 1;
            float2 g[2][4];
            slot_vector<DT>(from_g, 0, 32 * jj, g[0]);
            slot_vector<DT>(from_g, 1, half * 4 + 32 * jj, g[1]);
            if (HAD) row_hadamard<LANES>(g, j, lanes);
            if constexpr (MODE == kPairsHalves) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint4 c = load_shared16(turns + 16 * i), sn = load_shared16(turns + half * 4 + 16 * i);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float2 ce = make_float2(__uint_as_float(e ? c.z : c.x), __uint_as_float(e ? c.w : c.y));
                        const float2 se = make_float2(__uint_as_float(e ? sn.z : sn.x), __uint_as_float(e ? sn.w : sn.y));
                        const float2 u = g[0][2 * i + e], v = g[1][2 * i + e];
                        g[0][2 * i + e] = sub2(mul2(u, ce), mul2(v, se));
                        g[1][2 * i + e] = fma2(v, ce, mul2(u, se));
                    }
                }
            } else {
                row_rotate(g, turn, MODE, partner, jj, D, a.pairs);
            }
            float2 q = make_float2(0.f, 0.f), d = make_float2(0.f, 0.f);
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                float2 x[4];
                slot_vector<DT>(from_x, s, s * half * 4 + 32 * jj, x);
#pragma unroll
                for (int i = 0; i < 4; ++i) q = fma2(x[i], x[i], q);
            }
            const float sum = row_sum<LANES>(j < lanes ? q.x + q.y : 0.f);
            const float r = rsqrtf(sum * inv_d + a.eps), rc = r * hc;
            // dw += g h with h = x r; then g becomes g w
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                float2 x[4];
                slot_vector<DT>(from_x, s, s * half * 4 + 32 * jj, x);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float4 f = row_weights(wts, s, i, jj, lanes);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float2 &gi = g[s][2 * i + e];
                        const float2 xi = x[2 * i + e];
                        if (on) dw[s][2 * i + e] = fma2(mul2(gi, xi), make_float2(rc, rc), dw[s][2 * i + e]);
                        gi = mul2(gi, e ? make_float2(f.z, f.w) : make_float2(f.x, f.y));
                        d = fma2(xi, gi, d);
                    }
                }
            }
            const float dot = row_sum<LANES>(j < lanes ? d.x + d.y : 0.f);
            // dx = r (gw - h mean(gw h)) = r gw - x r^3 mean(gw x)
            const float k = -(r * r) * (rc * dot * inv_d);
            if (on) {
#pragma unroll
                for (int s = 0; s < 2; ++s) {
                    float2 x[4];
                    slot_vector<DT>(from_x, s, s * half * 4 + 32 * jj, x);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        g[s][i] = fma2(x[i], make_float2(k, k), mul2(g[s][i], make_float2(rc, rc)));
                }
                row_store<DT>(y, half * SIZE, g);
            }
            y += y_step;
            left -= per;
        }
    }
    asm volatile("cp.async.wait_group 0;\n" ::: "memory");

    __syncthreads();
    float *rows = (float *)smem;
    if (j < lanes)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) *(float2 *)(rows + group * D + s * half + 8 * j + 2 * i) = dw[s][i];
    __syncthreads();
    for (int i = threadIdx.x; i < D; i += kRowThreads) {
        float sum = 0.f;
        for (int w = 0; w < GROUPS; ++w) sum += rows[w * D + i];
        a.partial[(long long)blockIdx.x * D + i] = sum;
    }
}

// dw[i] = sum of the blocks' rows, in a fixed order: 32 warps take every 32nd row of 32 columns, then the warps are
// added in order.  blockIdx.y: queries or keys.  (Eight warps took 6 us longer: each row is a trip to L2.)
constexpr int kSumWarps = 32;
template <int DT>
__global__ void __launch_bounds__(32 * kSumWarps)
norm_weight_grad_kernel(const float *partial, int q_blocks, int k_blocks, int D, void *dwq, void *dwk, int w_f32)
{
    __shared__ float part[kSumWarps][32];
    pdl_launch_dependents();
    pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int i = blockIdx.x * 32 + lane;
    const float *rows = partial + (blockIdx.y ? (long long)q_blocks * D : 0);
    const int n = blockIdx.y ? k_blocks : q_blocks;
    float s = 0.f;
    if (i < D)
#pragma unroll 8
        for (int r = warp; r < n; r += kSumWarps) s += rows[(long long)r * D + i];
    part[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && i < D) {
        s = 0.f;
#pragma unroll
        for (int w = 0; w < kSumWarps; ++w) s += part[w][lane];
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

// Blocks of the gradient kernel that serve the queries and the keys: shares of the work, at least one each where there
// is any.  `most` bounds the sum (the size of the workspace goes by it).
struct GradBlocks {
    int q, k;
};
static GradBlocks grad_blocks(double q_work, double k_work, double work_per_block, int most)
{
    const double want = (q_work + k_work) / work_per_block;
    const int n = want < most ? (int)want + 1 : most;
    GradBlocks b{0, 0};
    if (q_work > 0) {
        b.q = k_work > 0 ? (int)(n * (q_work / (q_work + k_work)) + 0.5) : n;
        if (b.q < 1) b.q = 1;
    }
    if (k_work > 0) b.k = n - b.q > 1 ? n - b.q : 1;
    return b;
}
// Blocks of a gradient launch at most (one more may come from rounding up).  They do not go by the device's number of
// SMs, so that the order of the sums is the same on each.
constexpr int kGradBlocks = 148 * 8;
constexpr int row_grad_blocks(int dtype) { return 148 * (dtype == B200HT_F32 ? 2 : 3); }   // one wave of resident blocks

static int check_rot_common(const RotArgs &a, int dtype, int flags, const unsigned char *axis_of_pair, int n_axes)
{
    if (dtype != B200HT_F16 && dtype != B200HT_BF16 && dtype != B200HT_F32) return B200HT_ERR_DTYPE;
    if (flags & ~(B200HT_ROT_INTERLEAVED | B200HT_ROT_HADAMARD | B200HT_ROT_INVERSE | B200HT_ROT_POS64 | B200HT_ROT_WEIGHT_F32))
        return B200HT_ERR_SIZE;
    if (a.tokens < 0 || a.t[0].heads < 0 || a.t[1].heads < 0) return B200HT_ERR_SIZE;
    // the kernels and their grids count tokens, and both tensors' heads together, in 32 bits, rounded up to a block's share
    constexpr int kMostRows = (1 << 30) - 1;
    if (a.tokens > kMostRows || a.t[0].heads > kMostRows || a.t[1].heads > kMostRows) return B200HT_ERR_SIZE;
    if (a.D < 2 || a.D > kMaxHeadDim || (a.D & 1) || a.pairs < 1 || 2 * a.pairs > a.D) return B200HT_ERR_SIZE;
    if ((flags & B200HT_ROT_HADAMARD) && !is_pow2((uint64_t)a.D)) return B200HT_ERR_SIZE;
    if (n_axes < 1 || n_axes > kMaxAxes || (n_axes > 1 && !axis_of_pair)) return B200HT_ERR_SIZE;
    if (axis_of_pair)
        for (int i = 0; i < a.pairs; ++i)
            if (axis_of_pair[i] >= n_axes) return B200HT_ERR_SIZE;
    return 0;
}
static void fill_rot_common(RotArgs &a, int flags, const unsigned char *axis_of_pair, int n_axes)
{
    a.n_axes = n_axes;
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

// The layout of the fast form, or -1 where a row does not fit it.
static int row_mode(const RotArgs &a, int dtype, bool grad)
{
    if (a.D % 16) return -1;
    const long long vec = dtype == B200HT_F32 ? 4 : 8;
    for (const RotTensor &t : a.t) {
        if (!t.heads) continue;
        if (!aligned16(t.x) || !aligned16(t.y) || t.x_tok % vec || t.x_head % vec || t.y_tok % vec || t.y_head % vec) return -1;
        if (grad && (!aligned16(t.g) || t.g_tok % vec || t.g_head % vec)) return -1;
    }
    if (a.interleaved) return kPairsNeighbour;
    if (2 * a.pairs == a.D) return kPairsHalves;
    return a.pairs % 8 == 0 && 4 * a.pairs <= a.D ? kPairsInFirstHalf : -1;
}

// Tokens of a block.  Few tokens: one, so that all SMs have a block.  Else as many as leave the fewest groups idle in
// the last step of each walk over the heads, with several rows a group to share cos and sin and the block's start.
static int row_tokens(int groups, int q_heads, int k_heads, int tokens)
{
    if (tokens <= 2 * sm_count()) return 1;
    int best = 1;
    double best_use = 0;
    for (int tb = 1; tb <= groups && tb <= 16; tb *= 2) {
        const int per = groups / tb, steps = (q_heads + per - 1) / per + (k_heads + per - 1) / per;
        if (steps > 12 && best_use > 0) break;
        const double use = (double)(q_heads + k_heads) / (per * (steps + 0.5));
        if (use > best_use) { best_use = use; best = tb; }
    }
    return best;
}

template <int DT, bool NORM, int LANES>
static int launch_rows(const RotArgs &a, bool had, int mode, cudaStream_t st)
{
    const int tb = row_tokens(kRowThreads / LANES, a.t[0].heads, a.t[1].heads, a.tokens);
    const size_t smem = (size_t)tb * (a.D / 2) * sizeof(float2) + (NORM ? (size_t)2 * a.D * sizeof(float) : 0);
    const dim3 grid((unsigned)((a.tokens + tb - 1) / tb)), block(kRowThreads);
    return had ? launch_pdl(rotary_row_kernel<DT, NORM, true, LANES>, grid, block, smem, st, a, tb, mode)
               : launch_pdl(rotary_row_kernel<DT, NORM, false, LANES>, grid, block, smem, st, a, tb, mode);
}

template <int DT, bool NORM>
static int launch_forward(const RotArgs &a, bool had, int dtype, cudaStream_t st)
{
    const int mode = row_mode(a, dtype, false);
    if (mode < 0) return launch_any<DT, NORM>(a, had, st);
    if (a.D <= 64) return launch_rows<DT, NORM, 4>(a, had, mode, st);
    if (a.D <= 128) return launch_rows<DT, NORM, 8>(a, had, mode, st);
    return launch_rows<DT, NORM, 16>(a, had, mode, st);
}
template <int DT>
static int launch_rotary(const RotArgs &a, bool norm, bool had, cudaStream_t st)
{
    return norm ? launch_forward<DT, true>(a, had, DT, st) : launch_forward<DT, false>(a, had, DT, st);
}

template <int DT, int LANES, int MODE>
static int launch_row_grad_mode(const RotArgs &a, bool had, GradBlocks *b, cudaStream_t st)
{
    // groups of a warp for one token: all of them, fewer where the heads would leave some idle
    auto per = [](int heads) {
        int best = 32 / LANES, waste = 1 << 30;
        for (int p = 32 / LANES; p >= 1; p /= 2) {
            const int w = (heads + p - 1) / p * p - heads;
            if (w < waste) { waste = w; best = p; }
        }
        return best;
    };
    const int per_q = per(a.t[0].heads), per_k = per(a.t[1].heads);
    // a token costs its steps and, for cos and sin, about as much as one and a half more; a block has eight warps
    auto work = [&](int heads, int per) {
        return heads ? (double)a.tokens * (((heads + per - 1) / per) + 1.5) / (32 / LANES / per) : 0.;
    };
    const double q_work = work(a.t[0].heads, per_q), k_work = work(a.t[1].heads, per_k);
    *b = grad_blocks(q_work, k_work, kRowThreads / 32, row_grad_blocks(DT));
    if (b->q + b->k == 0) return 0;
    // the sums at the end ([groups][D] floats, 16 KB at most) take the place of the slots of rows (32 KB at least)
    const int tokens = 32 / LANES / (per_q < per_k ? per_q : per_k);
    const size_t smem = kRowSlots * row_slot_bytes<DT>() + (size_t)(kRowThreads / 32) * tokens * (a.D / 2) * sizeof(float2);
    const int rc = had ? ensure_dyn_smem((const void *)norm_rotary_row_grad_kernel<DT, true, LANES, MODE>, (int)smem)
                       : ensure_dyn_smem((const void *)norm_rotary_row_grad_kernel<DT, false, LANES, MODE>, (int)smem);
    if (rc) return rc;
    const dim3 grid((unsigned)(b->q + b->k)), block(kRowThreads);
    return had ? launch_pdl(norm_rotary_row_grad_kernel<DT, true, LANES, MODE>, grid, block, smem, st, a, per_q, per_k, b->q)
               : launch_pdl(norm_rotary_row_grad_kernel<DT, false, LANES, MODE>, grid, block, smem, st, a, per_q, per_k, b->q);
}

template <int DT, int LANES>
static int launch_row_grad(const RotArgs &a, bool had, int mode, GradBlocks *b, cudaStream_t st)
{
    if (mode == kPairsHalves) return launch_row_grad_mode<DT, LANES, kPairsHalves>(a, had, b, st);
    if (mode == kPairsNeighbour) return launch_row_grad_mode<DT, LANES, kPairsNeighbour>(a, had, b, st);
    return launch_row_grad_mode<DT, LANES, kPairsInFirstHalf>(a, had, b, st);
}

template <int DT>
static int launch_norm_grad(RotArgs &a, bool had, void *dwq, void *dwk, cudaStream_t st)
{
    const int mode = row_mode(a, DT, true);
    a.inverse = 1;
    GradBlocks b{0, 0};
    int rc = 0;
    if (mode < 0) {
        b = grad_blocks((double)a.tokens * a.t[0].heads, (double)a.tokens * a.t[1].heads, kAnyWarps, kGradBlocks);
        if (b.q + b.k) {
            const dim3 grid((unsigned)(b.q + b.k)), block(32 * kAnyWarps);
            rc = had ? launch_pdl(norm_rotary_any_grad_kernel<DT, true>, grid, block, 0, st, a, b.q)
                     : launch_pdl(norm_rotary_any_grad_kernel<DT, false>, grid, block, 0, st, a, b.q);
        }
    } else if (a.D <= 64) {
        rc = launch_row_grad<DT, 4>(a, had, mode, &b, st);
    } else if (a.D <= 128) {
        rc = launch_row_grad<DT, 8>(a, had, mode, &b, st);
    } else {
        rc = launch_row_grad<DT, 16>(a, had, mode, &b, st);
    }
    if (rc) return rc;
    return launch_pdl(norm_weight_grad_kernel<DT>, dim3((unsigned)((a.D + 31) / 32), 2), dim3(32 * kSumWarps), 0, st, (const float *)a.partial,
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
    fill_rot_common(a, flags, axis_of_pair, n_axes);
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
    fill_rot_common(a, flags, axis_of_pair, n_axes);
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
