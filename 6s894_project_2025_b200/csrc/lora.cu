// Low-rank adapters of many requests beside the shared projection:
//     C[m, t] = sum_k W[m, k] * (scale * H_K (d * x_t))[k]  +  s_a * sum_r B_a[m, r] * (sum_k A_a[r, k] * x_t[k]),
// a = index[t] the adapter of token t (none where it lies outside 0 .. adapters - 1).  The adapter sees the token as the
// caller gives it, without H: an adapter trained beside the unrotated weight keeps its matrices.
//
//   S = s_a * A_a x_t     lora_shrink_rows_kernel (few tokens: a block per token and some rows of A) or
//                         lora_shrink_tile_kernel (tcgen05: 128 tokens against the adapters among them)
//   C = W . H(X) + B S    prompts: further K steps of the contraction itself (gemm_tcgen05.cu), one rounding;
//                         decoding: fused GEMV into fp32, then lora_expand_kernel adds B S and rounds
// Sums are fp32; S is rounded to bf16 where it becomes an operand of the tensor cores (like H(X) itself), and stays fp32
// when decoding.  There is no counterpart in the reference.
#include "lora.cuh"
#include "tc_common.cuh"

namespace b200ht {

int launch_fwht(const void *in, void *out, uint64_t rows, uint32_t n, int dtype, float scale, const void *signs,
                cudaStream_t st, int keep_out);
int encode_tmap_bf16_stack(CUtensorMap *map, const void *base, uint64_t d2, uint64_t d1, uint64_t d0, uint32_t box1);
int fused_gemm_bf16_lora(const void *X, const void *W, void *C, int M, int N, int K, int out_dtype, int out_layout, float scale,
                         const void *signs, void *workspace, cudaStream_t st, const LoraGemm &lora);

// ---------------------------------------------------------------------------
// Which adapters occur in each tile of tokens.  A token whose adapter no earlier token of the tile has opens its entry
// in the list; the search goes backwards, so that a token next to one of its own request stops at once.
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(256) lora_plan_kernel(const int *index, int tokens, int adapters, int *tiles)
{
    __shared__ int ids[256];
    __shared__ int opened[2][8];
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long t = (long long)blockIdx.x * 256 + tid;
    int id = t < tokens ? index[t] : -1;
    if ((unsigned)id >= (unsigned)adapters) id = -1;
    ids[tid] = id;
    __syncthreads();
    bool first = id >= 0, first_half = first;
    for (int j = tid - 1; j >= 0 && first; --j)
        if (ids[j] == id) {
            first = false;
            if (j >= (tid & 128)) first_half = false;
        }
    const unsigned b = __ballot_sync(0xffffffffu, first), bh = __ballot_sync(0xffffffffu, first_half);
    if (lane == 0) {
        opened[0][warp] = __popc(b);
        opened[1][warp] = __popc(bh);
    }
    __syncthreads();
    int at = __popc(b & ((1u << lane) - 1)), at_half = __popc(bh & ((1u << lane) - 1));
    for (int w = 0; w < warp; ++w) at += opened[0][w];
    for (int w = warp & 4; w < warp; ++w) at_half += opened[1][w];
    int *tile = tiles + (size_t)blockIdx.x * kLoraTileInts;
    int *half = tile + kLoraHalfOffset + (tid >> 7) * kLoraHalfInts;
    if (first) tile[1 + at] = id;
    if (first_half) half[1 + at_half] = id;
    if (tid == 0) {
        int n = 0;
        for (int w = 0; w < 8; ++w) n += opened[0][w];
        tile[0] = n;
    }
    if ((tid & 127) == 0) {
        int n = 0;
        for (int w = warp; w < warp + 4; ++w) n += opened[1][w];
        half[0] = n;
    }
}

// ---------------------------------------------------------------------------
// S of few tokens: blockIdx.x the token, blockIdx.y a group of `rows` rows of its A; 8 / rows warps share a row.  Bound:
// the bytes of A (rank * K * 2 a token; tokens of one adapter share them through L2).  x comes from global memory where
// its elements are contiguous, else (b fastest, more than one column) through shared memory.
// ---------------------------------------------------------------------------
template <bool CONTIGUOUS, typename OUT>
__global__ void __launch_bounds__(256)
lora_shrink_rows_kernel(const __nv_bfloat16 *X, const __nv_bfloat16 *A, const int *index, const float *scaling, OUT *S, int tokens,
                        int K, int adapters, int rank, int rows)
{
    extern __shared__ __align__(16) __nv_bfloat16 xs[];
    __shared__ float part[8];
    pdl_launch_dependents();
    pdl_wait();
    const int t = blockIdx.x, r0 = blockIdx.y * rows;
    const int a = index[t];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int share = 8 / rows, r = r0 + warp / share;   // warps of a row; this warp's row
    const bool some = (unsigned)a < (unsigned)adapters;
    if (!CONTIGUOUS && some)
        for (int k = threadIdx.x; k < K; k += 256) xs[k] = X[(size_t)k * tokens + t];
    __syncthreads();
    float acc = 0.f;
    if (some && r < rank) {
        const uint4 *av = (const uint4 *)(A + ((size_t)a * rank + r) * K);
        const uint4 *xv = CONTIGUOUS ? (const uint4 *)(X + (size_t)t * K) : (const uint4 *)xs;
#pragma unroll 4
        for (int v = (warp % share) * 32 + lane; v < K / 8; v += share * 32) {
            const uint4 p = av[v], q = xv[v];
            const uint32_t pw[4] = {p.x, p.y, p.z, p.w}, qw[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 u = unpack2<B200HT_BF16>(pw[i]), w = unpack2<B200HT_BF16>(qw[i]);
                acc = fmaf(u.x, w.x, fmaf(u.y, w.y, acc));
            }
        }
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    if (lane == 0) part[warp] = acc;
    __syncthreads();
    if (threadIdx.x < rows && r0 + (int)threadIdx.x < rank) {
        float s = 0.f;
        for (int w = 0; w < share; ++w) s += part[threadIdx.x * share + w];
        if (some && scaling) s *= scaling[a];
        OUT *o = S + (size_t)t * rank + r0 + threadIdx.x;
        if constexpr (sizeof(OUT) == 4) *o = s;
        else *o = __float2bfloat16_rn(s);
    }
}

// ---------------------------------------------------------------------------
// Y = base + B S for a decoding batch.  A block takes 32 rows m of all columns: rank / 8 lanes (to a power of two) read a
// row of B_a as 16-byte vectors, so a warp reads consecutive rows of one adapter's B; the sums meet in shared memory in
// the layout of Y (b fastest) and leave with the fp32 base in one rounding.  Bound: the bytes of B.
// ---------------------------------------------------------------------------
constexpr int kExpandRows = 32;
__global__ void __launch_bounds__(256)
lora_expand_kernel(const float *base, const __nv_bfloat16 *B, const float *S, const int *index, void *Y, int M, int columns,
                   int adapters, int rank, int lanes, int out_dtype)
{
    extern __shared__ float sums[];   // [kExpandRows][columns]
    pdl_launch_dependents();
    pdl_wait();
    const int m0 = blockIdx.x * kExpandRows, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int j = lane % lanes, sub = lane / lanes, step = 32 / lanes;
    for (int t = warp; t < columns; t += 8) {
        const int a = index[t];
        const bool some = (unsigned)a < (unsigned)adapters;
        float s[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = some && 8 * j < rank ? S[(size_t)t * rank + 8 * j + i] : 0.f;
#pragma unroll 4
        for (int r = 0; r < kExpandRows; r += step) {
            const int m = m0 + r + sub;
            float acc = 0.f;
            if (some && m < M && 8 * j < rank) {
                const uint4 v = *(const uint4 *)(B + ((size_t)a * M + m) * rank + 8 * j);
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float2 u = unpack2<B200HT_BF16>(w[i]);
                    acc = fmaf(u.x, s[2 * i], fmaf(u.y, s[2 * i + 1], acc));
                }
            }
            for (int o = lanes / 2; o; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
            if (j == 0) sums[(r + sub) * columns + t] = acc;
        }
    }
    __syncthreads();
    const size_t at = (size_t)m0 * columns;
    const int n = (M - m0 < kExpandRows ? M - m0 : kExpandRows) * columns;
    for (int i = threadIdx.x; i < n; i += 256) {
        const float v = base[at + i] + sums[i];
        if (out_dtype == B200HT_F32) ((float *)Y)[at + i] = v;
        else ((__nv_bfloat16 *)Y)[at + i] = __float2bfloat16_rn(v);
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
template <typename OUT>
static int launch_shrink_rows(const void *X, const void *A, const int *index, const float *scaling, OUT *S, int tokens, int K,
                              int adapters, int rank, bool contiguous, cudaStream_t st)
{
    // one row of A a block spreads a short call over the SMs; with enough tokens eight rows share the block's start
    int rows = 8;
    while (rows > 1 && (long)tokens * ((rank + rows - 1) / rows) < 2 * sm_count()) rows /= 2;
    const dim3 grid((unsigned)tokens, (unsigned)((rank + rows - 1) / rows));
    if (contiguous)
        return launch_pdl(lora_shrink_rows_kernel<true, OUT>, grid, dim3(256), 0, st, (const __nv_bfloat16 *)X, (const __nv_bfloat16 *)A,
                          index, scaling, S, tokens, K, adapters, rank, rows);
    const size_t smem = (size_t)K * 2;
    int rc = ensure_dyn_smem((const void *)lora_shrink_rows_kernel<false, OUT>, (int)smem);
    if (rc) return rc;
    return launch_pdl(lora_shrink_rows_kernel<false, OUT>, grid, dim3(256), smem, st, (const __nv_bfloat16 *)X,
                      (const __nv_bfloat16 *)A, index, scaling, S, tokens, K, adapters, rank, rows);
}

static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

static int check_lora(int M, int N, int K, int adapters, int rank, int out_dtype)
{
    if (out_dtype != B200HT_F32 && out_dtype != B200HT_BF16) return B200HT_ERR_DTYPE;
    if (K < 64 || K > (1 << kMaxLogN) || !is_pow2((uint64_t)K)) return B200HT_ERR_SIZE;
    if (M < 0 || N < 0 || adapters < 1) return B200HT_ERR_SIZE;
    if (rank < 8 || rank > kLoraMaxRank || rank % 8) return B200HT_ERR_SIZE;
    return 0;
}

}  // namespace b200ht

extern "C" size_t b200ht_lora_gemm_workspace_bytes(int M, int N, int K, int rank)
{
    using namespace b200ht;
    if (M <= 0 || N <= 0 || K <= 0 || rank <= 0) return 0;
    return b200ht_fused_gemm_workspace_bytes(M, N, K, B200HT_BF16) + up256((size_t)N * rank * 2) +
           up256(((size_t)N + 255) / 256 * kLoraTileInts * sizeof(int));
}

extern "C" int b200ht_lora_gemm(const void *X, const void *W, void *C, const void *A, const void *B, const int *index,
                                const float *scaling, int M, int N, int K, int adapters, int rank, int out_dtype, int out_layout,
                                float scale, const void *signs, void *workspace, size_t workspace_bytes, void *stream)
{
    using namespace b200ht;
    int rc = check_lora(M, N, K, adapters, rank, out_dtype);
    if (rc) return rc;
    if (out_layout != B200HT_OUT_MN && out_layout != B200HT_OUT_NM) return B200HT_ERR_SIZE;
    if (M == 0 || N == 0) return 0;
    if (!X || !W || !C || !A || !B || !index) return B200HT_ERR_NULL;
    if (!aligned16(X) || !aligned16(W) || !aligned16(C) || !aligned16(A) || !aligned16(B) || (signs && !aligned16(signs)) ||
        ((uintptr_t)index & 3u) || ((uintptr_t)scaling & 3u))
        return B200HT_ERR_ALIGN;
    if (!workspace || workspace_bytes < b200ht_lora_gemm_workspace_bytes(M, N, K, rank)) return B200HT_ERR_WORKSPACE;
    if ((uintptr_t)workspace & 255u) return B200HT_ERR_ALIGN;
    rc = check_device();
    if (rc) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    unsigned char *ws = (unsigned char *)workspace + b200ht_fused_gemm_workspace_bytes(M, N, K, B200HT_BF16);
    __nv_bfloat16 *S = (__nv_bfloat16 *)ws;
    int *tiles = (int *)(ws + up256((size_t)N * rank * 2));
    const unsigned ntiles = (unsigned)((N + 255L) / 256);
    rc = launch_pdl(lora_plan_kernel, dim3(ntiles), dim3(256), 0, st, index, N, adapters, tiles);
    if (rc) return rc;
    rc = launch_shrink_rows(X, A, index, scaling, S, N, K, adapters, rank, true, st);
    if (rc) return rc;
    const LoraGemm lora{B, S, tiles, index, adapters, M, rank, 0};
    return fused_gemm_bf16_lora(X, W, C, M, N, K, out_dtype, out_layout, scale, signs, workspace, st, lora);
}

extern "C" size_t b200ht_lora_gemv_workspace_bytes(int M, int B, int rank)
{
    using namespace b200ht;
    if (M <= 0 || B <= 0 || rank <= 0) return 0;
    return up256((size_t)M * B * sizeof(float)) + up256((size_t)B * rank * sizeof(float));
}

extern "C" int b200ht_lora_gemv(const void *W, const void *X, void *Y, const void *A, const void *Bm, const int *index,
                                const float *scaling, int M, int N, int B, int adapters, int rank, int out_dtype, float scale,
                                void *workspace, size_t workspace_bytes, void *stream)
{
    using namespace b200ht;
    int rc = check_lora(M, B, N, adapters, rank, out_dtype);
    if (rc) return rc;
    if (B < 1 || B > 64) return B200HT_ERR_SIZE;
    if (M == 0) return 0;
    if (!W || !X || !Y || !A || !Bm || !index) return B200HT_ERR_NULL;
    if (!aligned16(W) || !aligned16(X) || !aligned16(Y) || !aligned16(A) || !aligned16(Bm) || ((uintptr_t)index & 3u) ||
        ((uintptr_t)scaling & 3u))
        return B200HT_ERR_ALIGN;
    if (!workspace || workspace_bytes < b200ht_lora_gemv_workspace_bytes(M, B, rank)) return B200HT_ERR_WORKSPACE;
    if ((uintptr_t)workspace & 255u) return B200HT_ERR_ALIGN;
    rc = check_device();
    if (rc) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    float *base = (float *)workspace, *S = (float *)((unsigned char *)workspace + up256((size_t)M * B * sizeof(float)));
    rc = launch_shrink_rows(X, A, index, scaling, S, B, N, adapters, rank, B == 1, st);
    if (rc) return rc;
    rc = b200ht_fused_gemv(W, X, base, M, N, B, B200HT_BF16, B200HT_F32, scale, stream);
    if (rc) return rc;
    int lanes = 1;
    while (lanes * 8 < rank) lanes *= 2;
    return launch_pdl(lora_expand_kernel, dim3((unsigned)((M + kExpandRows - 1) / kExpandRows)), dim3(256),
                      (size_t)kExpandRows * B * sizeof(float), st, (const float *)base, (const __nv_bfloat16 *)Bm, (const float *)S,
                      index, Y, M, B, adapters, rank, lanes, out_dtype);
}
