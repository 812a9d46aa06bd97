// Low-rank adapters of many requests beside the shared projection:
//     C[m, t] = sum_k W[m, k] * (scale * H_K (d * x_t))[k]  +  s_a * sum_r B_a[m, r] * (sum_k A_a[r, k] * x_t[k]),
// a = index[t] the adapter of token t (none where it lies outside 0 .. adapters - 1).  The adapter sees the token as the
// caller gives it, without H: an adapter trained beside the unrotated weight keeps its matrices.
//
//   H(X)                  lora_transform_kernel: fp32 throughout, one rounding to bf16
//   S = s_a * A_a x_t     lora_shrink_rows_kernel (few tokens: a block per token and some rows of A) or
//                         lora_shrink_tile_kernel (tcgen05: 256 tokens against the adapters among them)
//   C = W . H(X) + B S    prompts: further K steps of the contraction itself (gemm_tcgen05.cu), one rounding;
//                         decoding: lora_front_kernel (H(X) and S in one launch), then the streaming GEMV, which adds
//                         B S to its sums (fused_gemv.cu); shapes that do not take it: fused GEMV into fp32, then
//                         lora_expand_kernel adds B S and rounds
// Sums are fp32; S is rounded to bf16 where it becomes an operand of the tensor cores (like H(X) itself), and stays fp32
// when decoding.  There is no counterpart in the reference.
#include <type_traits>

#include "lora_tc.cuh"

namespace b200ht {

int launch_gemv_adapt(const void *W, const void *Xt, void *Y, int M, int N, int B, int out_dtype, const GemvAdapt &adapt,
                      cudaStream_t st);
bool gemv_adapt_shape(int N, int B);
int fused_gemm_bf16_lora(const void *X, const void *W, void *C, int M, int N, int K, int out_dtype, int out_layout, float scale,
                         const void *signs, void *workspace, cudaStream_t st, const LoraGemm &lora);

// ---------------------------------------------------------------------------
// Which adapters occur among 256 tokens.  Called by 256 threads, eight warps, with the token's adapter (-1: none); a token
// whose adapter no earlier one has opens an entry.  Earlier tokens of its warp are found by a match; only a warp's first
// token of an adapter looks through the warps before, four tokens a load.
// ---------------------------------------------------------------------------
struct TileAdapters {
    __align__(16) int ids[256];
    int entry[256];      // entry of the adapter that this token opened
    int opened[8];
};
// Returns the number of entries; `mine`: this token's, `first`: it opened it.  `sync` is a barrier of the 256 threads.
template <typename Sync>
__device__ __forceinline__ int tile_adapters(TileAdapters &t, int tid, int id, int &mine, bool &first, Sync sync)
{
    const int lane = tid & 31, warp = tid >> 5;
    t.ids[tid] = id;
    const unsigned alike = __match_any_sync(0xffffffffu, id);   // by all lanes: not behind a condition
    sync();
    int earliest = tid;
    if (id >= 0 && (alike & ((1u << lane) - 1)) == 0) {
        const int4 *four = (const int4 *)t.ids;
#pragma unroll 4
        for (int j = warp * 8 - 1; j >= 0; --j) {
            const int4 v = four[j];
            if (v.w == id) earliest = 4 * j + 3;
            if (v.z == id) earliest = 4 * j + 2;
            if (v.y == id) earliest = 4 * j + 1;
            if (v.x == id) earliest = 4 * j;
        }
    }
    earliest = __shfl_sync(0xffffffffu, earliest, __ffs(alike) - 1);
    first = id >= 0 && earliest == tid;
    const unsigned b = __ballot_sync(0xffffffffu, first);
    if (lane == 0) t.opened[warp] = __popc(b);
    sync();
    int at = __popc(b & ((1u << lane) - 1)), n = 0;
    for (int w = 0; w < 8; ++w) {
        if (w < warp) at += t.opened[w];
        n += t.opened[w];
    }
    if (first) t.entry[tid] = at;
    sync();
    mine = id >= 0 ? t.entry[earliest] : -1;
    return n;
}

// The tables of the tiles (lora.cuh).
__global__ void __launch_bounds__(256) lora_plan_kernel(const int *index, int tokens, int adapters, int *tiles)
{
    __shared__ TileAdapters found;
    __shared__ unsigned own[256][8];
    pdl_wait();
    pdl_launch_dependents();   // the rest of the chain starts after all earlier work: its kernels may read inputs at once
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const long long t = (long long)blockIdx.x * 256 + tid;
    int id = t < tokens ? index[t] : -1;
    if ((unsigned)id >= (unsigned)adapters) id = -1;
#pragma unroll
    for (int w = 0; w < 8; ++w) own[tid][w] = 0;
    int mine;
    bool first;
    const int n = tile_adapters(found, tid, id, mine, first, [] { __syncthreads(); });
    int *tile = tiles + (size_t)blockIdx.x * kLoraTileInts;
    if (first) tile[1 + mine] = id;
    if (tid == 0) tile[0] = n;
    const unsigned valid = __ballot_sync(0xffffffffu, id >= 0);
    if (lane == 0) tile[kLoraValidOffset + warp] = (int)valid;
    if (id >= 0) atomicOr(&own[mine][warp], 1u << lane);
    __syncthreads();
    for (int i = tid; i < n * 8; i += 256) tile[kLoraOwnOffset + i] = (int)own[i >> 3][i & 7];
}

// ---------------------------------------------------------------------------
// H of one token by one block, in fp32 with one rounding at the end (the transform of fwht.cu passes 16-bit values between
// its stages, two or three roundings more; beside adapters, whose share of the result is small, they would be the larger
// error).  The row lies in shared memory as fp32 lines of 32 values, their 16-byte pieces exchanged by the line's number
// so that no access below meets bank conflicts:
//   A  32 consecutive values a thread from global memory: bits 0 .. 4 of the index
//   B  rounds of up to five bits from bit 5 on, lanes side by side (one for K = 8192, two beyond)
//   C  8 consecutive values and the last three bits: scaled, rounded, stored as 16-byte vectors
// Bound: shared memory and the instruction rate (0.63 issued a cycle): 2048 tokens of 8192 in 19 us (10 at the copy
// bandwidth, fwht.cu 12); with the places computed element by element 32 us.
// ---------------------------------------------------------------------------
__device__ __forceinline__ int line_at(int e)   // place of element e
{
    const int line = e >> 5;
    return (line << 5) | ((((e >> 2) ^ line) & 7) << 2) | (e & 3);
}
// `bit` and the sizes are constants, so that the places of a thread's elements differ by constants: in the line's number
// by multiples of 2^(bit - 5), which exchange pieces only in its low three bits.
template <int BITS, int BIT, int K>
__device__ __forceinline__ void fwht_round(float *row)   // bits BIT .. BIT + BITS - 1, BIT >= 5
{
    for (int task = threadIdx.x; task < (K >> BITS); task += blockDim.x) {
        const int at = line_at(((task >> BIT) << (BIT + BITS)) | (task & ((1 << BIT) - 1)));
        float v[1 << BITS];
#pragma unroll
        for (int i = 0; i < (1 << BITS); ++i) v[i] = row[(at ^ (((i << (BIT - 5)) & 7) << 2)) + (i << BIT)];
#pragma unroll
        for (int m = 1; m < (1 << BITS); m <<= 1)
#pragma unroll
            for (int i = 0; i < (1 << BITS); ++i)
                if (!(i & m)) {
                    const float a = v[i], b = v[i | m];
                    v[i] = a + b;
                    v[i | m] = a - b;
                }
#pragma unroll
        for (int i = 0; i < (1 << BITS); ++i) row[(at ^ (((i << (BIT - 5)) & 7) << 2)) + (i << BIT)] = v[i];
    }
    __syncthreads();
}
template <int BITS, int K>
__device__ __forceinline__ void fwht_last(const float *row, __nv_bfloat16 *out, float scale)
{
    constexpr int N = 1 << BITS, STEP = K >> BITS;
    for (int task = threadIdx.x; task < STEP / 8; task += blockDim.x) {
        float v[N][8];
        const int at0 = line_at(task * 8), at1 = line_at(task * 8 + 4);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            constexpr int LINES = STEP / 32;   // from one of the N pieces to the next
            const int x = ((i * LINES) & 7) << 2;
            const float4 f = *(const float4 *)(row + (LINES % 8 ? line_at(task * 8 + i * STEP) : (at0 ^ x) + i * STEP));
            const float4 g = *(const float4 *)(row + (LINES % 8 ? line_at(task * 8 + i * STEP + 4) : (at1 ^ x) + i * STEP));
            v[i][0] = f.x, v[i][1] = f.y, v[i][2] = f.z, v[i][3] = f.w, v[i][4] = g.x, v[i][5] = g.y, v[i][6] = g.z, v[i][7] = g.w;
        }
#pragma unroll
        for (int m = 1; m < N; m <<= 1)
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (!(i & m))
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float a = v[i][e], b = v[i | m][e];
                        v[i][e] = a + b;
                        v[i | m][e] = a - b;
                    }
#pragma unroll
        for (int i = 0; i < N; ++i)
            *(uint4 *)(out + task * 8 + i * STEP) =
                make_uint4(pack2<B200HT_BF16>(v[i][0] * scale, v[i][1] * scale), pack2<B200HT_BF16>(v[i][2] * scale, v[i][3] * scale),
                           pack2<B200HT_BF16>(v[i][4] * scale, v[i][5] * scale), pack2<B200HT_BF16>(v[i][6] * scale, v[i][7] * scale));
    }
}
// K = 2^LOGK >= 64; x: the token's values, contiguous; out: K values; signs: 0x8000 where an element is negated, or NULL.
template <int LOGK>
__device__ __forceinline__ void fwht_token(float *row, const __nv_bfloat16 *x, __nv_bfloat16 *out, float scale, const uint16_t *signs)
{
    constexpr int K = 1 << LOGK, LAST = LOGK - 5 < 3 ? LOGK - 5 : 3, MIDDLE = LOGK - 5 - LAST;
    for (int task = threadIdx.x; task < K / 32; task += blockDim.x) {
        float v[32];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint4 p = ((const uint4 *)(x + task * 32))[i];
            if (signs) {
                const uint4 sg = ((const uint4 *)(signs + task * 32))[i];
                p.x ^= sg.x, p.y ^= sg.y, p.z ^= sg.z, p.w ^= sg.w;
            }
            const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 f = unpack2<B200HT_BF16>(w[e]);
                v[8 * i + 2 * e] = f.x;
                v[8 * i + 2 * e + 1] = f.y;
            }
        }
#pragma unroll
        for (int m = 1; m < 32; m <<= 1)
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (!(i & m)) {
                    const float a = v[i], b = v[i | m];
                    v[i] = a + b;
                    v[i | m] = a - b;
                }
#pragma unroll
        for (int i = 0; i < 8; ++i)
            *(float4 *)(row + line_at(task * 32 + 4 * i)) = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    }
    __syncthreads();
    if constexpr (MIDDLE > 5) {
        fwht_round<(MIDDLE + 1) / 2, 5, K>(row);
        fwht_round<MIDDLE / 2, 5 + (MIDDLE + 1) / 2, K>(row);
    } else if constexpr (MIDDLE > 0) {
        fwht_round<MIDDLE, 5, K>(row);
    }
    fwht_last<LAST, K>(row, out, scale);
}
// f(std::integral_constant<int, logk>) for logk = FROM .. 15.
template <int FROM, typename F>
static int with_logk(int logk, F f)
{
    if (logk == FROM) return f(std::integral_constant<int, FROM>{});
    if constexpr (FROM < kMaxLogN) return with_logk<FROM + 1>(logk, f);
    return B200HT_ERR_SIZE;
}

// `early`: X is complete and Y free as soon as this kernel starts (it follows lora_plan_kernel); it then runs beside the
// kernels in front and waits for them before it ends, so that whoever waits for it has waited for them too.
template <int LOGK>
__global__ void __launch_bounds__(256) lora_transform_kernel(const __nv_bfloat16 *X, __nv_bfloat16 *Y, float scale, const uint16_t *signs,
                                                             int early)
{
    extern __shared__ __align__(16) unsigned char smem_row[];
    pdl_launch_dependents();
    if (!early) pdl_wait();
    const size_t at = (size_t)blockIdx.x << LOGK;
    fwht_token<LOGK>((float *)smem_row, X + at, Y + at, scale, signs);
    if (early) pdl_wait();
}

// ---------------------------------------------------------------------------
// S of few tokens: a block takes `rows` rows of a token's A; 8 / rows warps share a row.  Bound: the bytes of A
// (rank * K * 2 a token; tokens of one adapter share them through L2).  x comes from global memory where its elements are
// contiguous, else (b fastest, more than one column) through shared memory.
// ---------------------------------------------------------------------------
template <typename OUT>
__device__ __forceinline__ void shrink_rows(const __nv_bfloat16 *X, int stride, size_t token_at, const __nv_bfloat16 *A, int a, bool some,
                                            const float *scaling, OUT *S, __nv_bfloat16 *xs, int K, int rank, int r0, int rows)
{   // `rank`: rows of A; S: the token's
    __shared__ float part[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int share = 8 / rows, r = r0 + warp / share;   // warps of a row; this warp's row
    if (stride != 1) {
        if (some)
#pragma unroll 8
            for (int k = threadIdx.x; k < K; k += 256) xs[k] = X[token_at + (size_t)k * stride];
        __syncthreads();
    }
    float acc = 0.f;
    if (some && r < rank) {
        const uint4 *av = (const uint4 *)(A + ((size_t)a * rank + r) * K);
        const uint4 *xv = stride == 1 ? (const uint4 *)(X + token_at) : (const uint4 *)xs;
#pragma unroll 8
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
        if constexpr (sizeof(OUT) == 4) S[r0 + threadIdx.x] = s;
        else S[r0 + threadIdx.x] = __float2bfloat16_rn(s);
    }
}

// stride: distance of two elements of a token; token t begins at t * (stride == 1 ? K : 1).  `early`: as in
// lora_transform_kernel.
template <typename OUT>
__global__ void __launch_bounds__(256)
lora_shrink_rows_kernel(const __nv_bfloat16 *X, int stride, const __nv_bfloat16 *A, const int *index, const float *scaling, OUT *S,
                        int K, int adapters, int rank, int rows, int early)
{
    extern __shared__ __align__(16) unsigned char smem_row[];
    pdl_launch_dependents();
    if (!early) pdl_wait();
    const int t = blockIdx.x, a = index[t];
    shrink_rows<OUT>(X, stride, (size_t)t * (stride == 1 ? K : 1), A, a, (unsigned)a < (unsigned)adapters, scaling,
                     S + (size_t)t * (sizeof(OUT) == 2 ? lora_pitch(rank) : rank), (__nv_bfloat16 *)smem_row, K, rank, blockIdx.y * rows, rows);
    if (early) pdl_wait();
}

// Decoding: H(X) and S of every column in one launch.  It lets the next kernel start only once it has itself seen all
// earlier work complete, so the streaming GEMV behind it may read W, B and index at once and waits for nothing but Xt and S.
//
// Tokens whose elements lie side by side (CLUSTER false; a single column too): the first blocks transform one each, the
// others take `rows` rows of a token's A, x comes straight from memory.
// Columns of a matrix: a cluster of eight CTAs a column.  The elements of a column lie a row of X apart, a 32-byte sector
// each, so every CTA fetches an eighth and they exchange it through distributed shared memory (each fetching all of it,
// 272 CTAs of a batch of 16 at N = 4096 moved 35 MB through L2 and took 8 us).  Rank 0 transforms, the others divide A.
template <bool CLUSTER, int LOGK>
__global__ void __launch_bounds__(256)
lora_front_kernel(const __nv_bfloat16 *X, const __nv_bfloat16 *A, const int *index, const float *scaling, __nv_bfloat16 *Xt, float *S,
                  int columns, float scale, int adapters, int rank, int rows)
{
    extern __shared__ __align__(16) unsigned char smem_row[];
    pdl_wait();
    pdl_launch_dependents();
    constexpr int K = 1 << LOGK;
    if constexpr (!CLUSTER) {
        if ((int)blockIdx.x < columns) {
            const size_t at = (size_t)blockIdx.x << LOGK;
            fwht_token<LOGK>((float *)smem_row, X + at, Xt + at, scale, nullptr);
        } else {
            const int groups = (rank + rows - 1) / rows, i = blockIdx.x - columns, t = i / groups, a = index[t];
            shrink_rows<float>(X, 1, (size_t)t << LOGK, A, a, (unsigned)a < (unsigned)adapters, scaling, S + (size_t)t * rank, nullptr, K,
                               rank, (i - t * groups) * rows, rows);
        }
        return;
    }
    __nv_bfloat16 *xs = (__nv_bfloat16 *)smem_row;   // the column; behind it the transform's fp32 row
    const int column = blockIdx.x / 8, part = blockIdx.x % 8, slice = K / 8;
    const int a = index[column];
    const __nv_bfloat16 *x = X + (size_t)part * slice * columns + column;
#pragma unroll 4
    for (int k = threadIdx.x; k < slice; k += 256) xs[part * slice + k] = x[(size_t)k * columns];
    cluster_sync_all();
    for (int v = threadIdx.x; v < K / 8; v += 256) {
        const int from = v / (slice / 8);
        if (from == part) continue;
        uint32_t at;
        uint4 p;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(at) : "r"(smem_u32(xs) + (uint32_t)v * 16), "r"(from));
        asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(p.x), "=r"(p.y), "=r"(p.z), "=r"(p.w) : "r"(at) : "memory");
        ((uint4 *)xs)[v] = p;
    }
    cluster_sync_all();   // no CTA writes again what others read, and none has left before they have
    if (part == 0) {
        fwht_token<LOGK>((float *)(smem_row + K * 2), xs, Xt + ((size_t)column << LOGK), scale, nullptr);
    } else {
        const int per = (rank + 6) / 7, r0 = (part - 1) * per, r1 = r0 + per < rank ? r0 + per : rank;
        const bool some = (unsigned)a < (unsigned)adapters;
        for (int r = r0; r < r1; r += rows) {
            shrink_rows<float>(xs, 1, 0, A + (some ? (size_t)a * rank * K : 0), 0, some, nullptr, S + (size_t)column * rank, nullptr, K, r1,
                               r, rows);
            __syncthreads();
        }
        if (some && scaling && (int)threadIdx.x < r1 - r0) S[(size_t)column * rank + r0 + threadIdx.x] *= scaling[a];
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
// S of many tokens, on the tensor cores: 256 tokens (the N of the instruction) against the A matrices of the adapters among
// them, 128 / rank of which share the M of one instruction, two such groups a pass; K is split over the CTAs of a cluster.
// Each token keeps the rows of its own adapter.  With prompts a tile has a few adapters, one pass serves them and X is read
// once; bound then: the bytes of X.  (Full instructions pay: with 128 tokens as M and an instruction an adapter, 16384 x
// 8192 tokens of 40 requests at rank 64 took 94 us; with the adapters as M and 128 tokens as N, 97 us, two tiles an SM
// taking turns and a second pass where a tile had three adapters; so 71 us, 41 at the copy bandwidth.)  Short prompts are bound by the chain of latencies: 2001 x 4096 at rank 32 takes 14 us.
//
// Warp 0 copies by TMA (X 256 x 64 and rank x 64 of each adapter's A a stage, 128-byte swizzle), warp 1 issues the MMAs,
// warps 2..9 find the tile's adapters while the first tiles of X arrive, and at the end bring the accumulators (one row of
// an A a lane) into shared memory, over the stages that have been used up.  The CTAs of the cluster then add the partial
// sums of 256 / cluster tokens each through distributed shared memory, in the order of the ranks, and write them with one
// rounding: no atomics, no partial sums in memory.
// The kernel runs beside lora_plan_kernel (its inputs are complete when it starts) and waits for it at its end.
// ---------------------------------------------------------------------------
constexpr int kShrinkStages = 3, kShrinkThreads = 320;
constexpr int kShrinkXBytes = 256 * 128, kShrinkStageBytes = 2 * kShrinkXBytes;
constexpr int kShrinkSmem = kShrinkStages * kShrinkStageBytes + 1024 + 128;
static_assert(256 * kLoraMaxRank * 4 <= kShrinkStages * kShrinkStageBytes, "the partial sums lie over the stages");

__device__ __forceinline__ float4 cluster_load4(uint32_t local, int rank)   // from `local` in the shared memory of CTA `rank`
{
    float4 v;
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(at) : "r"(local), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
    return v;
}

__global__ void __launch_bounds__(kShrinkThreads, 1)
lora_shrink_tile_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmA, const int *index,
                        const float *scaling, __nv_bfloat16 *S, int tokens, int adapters, int rank, int kblocks, int split, int *status)
{
    extern __shared__ unsigned char smem_dyn[];
    __shared__ TileAdapters found;
    __shared__ __align__(16) int list[256], slot[256];   // the tile's adapters; each token's place among them
    __shared__ float factor[256];          // scaling of each token's adapter
    __shared__ int count_s;
    const uint32_t base = (smem_u32(smem_dyn) + 1023u) & ~1023u;
    unsigned char *gen = smem_dyn + (base - smem_u32(smem_dyn));
    const uint32_t bars = base + kShrinkStages * kShrinkStageBytes;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (kShrinkStages + s); };
    const uint32_t done_bar = bars + 16u * kShrinkStages;
    uint32_t *tmem_slot = (uint32_t *)(gen + kShrinkStages * kShrinkStageBytes + 16 * kShrinkStages + 8);
    volatile int *abort_flag = (volatile int *)(tmem_slot + 1);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int part = blockIdx.x % split, tile = blockIdx.x / split;   // rank in the cluster, 256-token tile
    const int t0 = tile * 256;
    const int nk = kblocks / split, kb0 = part * nk, ahead = nk < kShrinkStages ? nk : kShrinkStages;

    if (tid == 0) {
        for (int s = 0; s < kShrinkStages; ++s) {
            mbar_init(full_bar(s), 2);   // X, the A matrices
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(done_bar, 1);
        *abort_flag = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tmX);
        tma_prefetch_desc(&tmA);
    }
    if (warp == 1) tmem_alloc(smem_u32(tmem_slot), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();   // not before this CTA has its TMEM: the contraction behind takes all of it

    auto load_x = [&](int s, int kb) {
        mbar_expect_tx(full_bar(s), (uint32_t)kShrinkXBytes);
        tma_load_3d(base + s * kShrinkStageBytes, &tmX, kb * 64, t0, 0, full_bar(s));
    };
    if (warp == 0) {
        if (lane == 0)
            for (int i = 0; i < ahead; ++i) load_x(i, kb0 + i);
        __syncwarp();
    } else if (warp >= 2) {
        const int t = tid - 64;
        int id = t0 + t < tokens ? __ldcg(index + t0 + t) : -1, mine;
        if ((unsigned)id >= (unsigned)adapters) id = -1;
        bool first;
        const float f = scaling && id >= 0 ? scaling[id] : 1.f;   // under way while the adapters are found
        const int n = tile_adapters(found, t, id, mine, first, [] { asm volatile("bar.sync 1, 256;\n" ::: "memory"); });
        slot[t] = mine;
        factor[t] = f;
        if (first) list[mine] = id;
        if (t == 0) count_s = n;
    }
    __syncthreads();
    const int count = count_s;
    const int share = 128 / rank;                   // adapters of one instruction
    float *partial = (float *)gen;                  // [256][rank], over the stages
    const int out_pitch = lora_pitch(rank);
    const int rows = 256 / split, row0 = part * rows;   // tokens whose sums this CTA writes
    if (blockIdx.y == 0)                            // tokens without an adapter
        for (int i = tid; i < rows * (rank / 8); i += kShrinkThreads) {
            const int row = row0 + i / (rank / 8);
            if (t0 + row < tokens && slot[row] < 0)
                *(uint4 *)(S + (size_t)(t0 + row) * out_pitch + i % (rank / 8) * 8) = make_uint4(0u, 0u, 0u, 0u);
        }

    int it = 0, passes = 0;   // K steps so far; X of the first `ahead` is on its way
    bool ok = true;           // once a wait has run out this CTA copies and multiplies no more, but keeps step with its cluster
    for (int first = blockIdx.y * 2 * share; first < count; first += gridDim.y * 2 * share, ++passes) {
        const int n = count - first < 2 * share ? count - first : 2 * share;   // adapters of this pass, `share` a group
        const int groups = n > share ? 2 : 1;
        if (!ok) {
        } else if (warp == 0 && lane == 0) {
            int i2 = it;
            for (int kb = kb0; kb < kb0 + nk; ++kb, ++i2) {
                const int s = i2 % kShrinkStages;
                if (i2 >= ahead) {
                    if (!mbar_wait(empty_bar(s), ((i2 / kShrinkStages) & 1u) ^ 1u, abort_flag, status)) { ok = false; break; }
                    load_x(s, kb);
                }
                mbar_expect_tx(full_bar(s), (uint32_t)(n * rank * 128));
                uint32_t to = base + s * kShrinkStageBytes + kShrinkXBytes;
                for (int a = 0; a < n; ++a) {
                    if (a == share) to = base + s * kShrinkStageBytes + kShrinkXBytes + 16384;
                    tma_load_3d(to, &tmA, kb * 64, 0, list[first + a], full_bar(s));
                    to += rank * 128;
                }
            }
            if (!ok) {   // copies on their way still land in this CTA's shared memory: give them time
                const int pending = i2 < kShrinkStages ? i2 : kShrinkStages;
                for (int j = 1; j <= pending; ++j) {
                    const uint64_t ns = global_ns();
                    while (!mbar_test(full_bar((i2 - j) % kShrinkStages), ((i2 - j) / kShrinkStages) & 1u) && global_ns() - ns < 100000000ull) {}
                }
            }
        } else if (warp == 1 && lane == 0) {
            constexpr uint32_t idesc = umma_idesc_bf16(128, 256);
            int i2 = it;
            for (int kb = 0; kb < nk; ++kb, ++i2) {
                const int s = i2 % kShrinkStages;
                if (!mbar_wait(full_bar(s), (i2 / kShrinkStages) & 1u, abort_flag, status)) { ok = false; break; }
                tc_fence_after();
                const uint32_t sa = base + s * kShrinkStageBytes;
                const uint64_t xdesc = umma_desc_k_sw128(sa);
                // rows of the A operand behind the adapters' hold whatever was there: their sums are not read
                for (int g = 0; g < groups; ++g) {
                    const uint64_t adesc = umma_desc_k_sw128(sa + kShrinkXBytes + g * 16384);
#pragma unroll
                    for (int k = 0; k < 4; ++k) umma_bf16_ss(tmem + g * 256, adesc + 2 * k, xdesc + 2 * k, idesc, (kb | k) ? 1u : 0u);
                }
                umma_commit(empty_bar(s));
            }
            if (ok) umma_commit(done_bar);
        }
        __syncwarp();
        it += nk;
        // all MMAs of the pass done: the accumulators are complete and the stages are free
        ok = __syncthreads_and(ok && mbar_wait(done_bar, passes & 1u, abort_flag, status));
        if (ok && warp >= 2) {
            tc_fence_after();
            const int q = warp & 3, row = q * 32 + lane, a = row / rank, r = row - a * rank;
            const int c0 = (warp - 2) / 4 * 128;   // two warps share the lanes of a quadrant
#pragma unroll 1
            for (int g = 0; g < groups; ++g) {
                const int mine = a < share && g * share + a < n ? first + g * share + a : -2;   // -2 is no token's place
#pragma unroll 1
                for (int c = c0; c < c0 + 128; c += 32) {
                    uint32_t v[32], keep = 0;   // bit i: token c + i is this adapter's
                    tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + g * 256 + c, v);
                    // all places before the first store, which would hold back the loads behind it
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int4 p = *(const int4 *)(slot + c + 4 * i);
                        keep |= (p.x == mine ? 1u : 0u) << (4 * i) | (p.y == mine ? 2u : 0u) << (4 * i) | (p.z == mine ? 4u : 0u) << (4 * i) |
                                (p.w == mine ? 8u : 0u) << (4 * i);
                    }
                    tmem_ld_wait();
                    float *to = partial + c * rank + r;
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if ((keep >> i) & 1u) to[i * rank] = __uint_as_float(v[i]);
                }
            }
            tc_fence_before();
        }
        cluster_sync_all();
        const int fours = rank / 4;
        for (int i = tid; i < rows * fours && ok; i += kShrinkThreads) {
            const int row = row0 + i / fours, r = i % fours * 4, mine = slot[row] - first;
            if (mine < 0 || mine >= n) continue;
            const uint32_t at = base + (uint32_t)((row * rank + r) * 4);
            float4 v[8], sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int p = 0; p < 8; ++p)
                if (p < split) v[p] = cluster_load4(at, p);
#pragma unroll
            for (int p = 0; p < 8; ++p)
                if (p < split) sum = make_float4(sum.x + v[p].x, sum.y + v[p].y, sum.z + v[p].z, sum.w + v[p].w);
            const float f = factor[row];
            *(uint2 *)(S + (size_t)(t0 + row) * out_pitch + r) = make_uint2(pack2<B200HT_BF16>(sum.x * f, sum.y * f), pack2<B200HT_BF16>(sum.z * f, sum.w * f));
        }
        fence_proxy_async();   // the next pass' copies overwrite what was read here
        cluster_sync_all();
    }
    if (passes == 0 && warp == 0 && lane == 0)   // nothing to do here, but X has been asked for: let it arrive
        for (int i = 0; i < ahead; ++i) {
            mbar_arrive(full_bar(i));
            mbar_wait(full_bar(i), 0u, abort_flag, status);
        }
    pdl_wait();
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
// Rows of A a block takes: one spreads a short call over the SMs; with enough tokens eight share the block's start.
static int shrink_rows_of_block(int tokens, int rank)
{
    int rows = 8;
    while (rows > 1 && (long)tokens * ((rank + rows - 1) / rows) < 2 * sm_count()) rows /= 2;
    return rows;
}

template <typename OUT>
static int launch_shrink_rows(const void *X, const void *A, const int *index, const float *scaling, OUT *S, int tokens, int K,
                              int adapters, int rank, int stride, bool early, cudaStream_t st)
{
    const int rows = shrink_rows_of_block(tokens, rank);
    const size_t smem = stride == 1 ? 0 : (size_t)K * 2;
    int rc = ensure_dyn_smem((const void *)lora_shrink_rows_kernel<OUT>, (int)smem);
    if (rc) return rc;
    return launch_pdl(lora_shrink_rows_kernel<OUT>, dim3((unsigned)tokens, (unsigned)((rank + rows - 1) / rows)), dim3(256), smem, st,
                      (const __nv_bfloat16 *)X, stride, (const __nv_bfloat16 *)A, index, scaling, S, K, adapters, rank, rows, early ? 1 : 0);
}

int launch_lora_transform(const void *X, void *Y, int tokens, int K, float scale, const void *signs, bool early, cudaStream_t st)
{
    const int threads = K / 64 < 64 ? 64 : (K / 64 > 256 ? 256 : K / 64), smem = K * 4;
    return with_logk<6>(ilog2((uint32_t)K), [&](auto logk) {
        const auto kernel = lora_transform_kernel<decltype(logk)::value>;
        int rc = ensure_dyn_smem((const void *)kernel, smem);
        if (rc) return rc;
        return launch_pdl(kernel, dim3((unsigned)tokens), dim3((unsigned)threads), (size_t)smem, st, (const __nv_bfloat16 *)X,
                          (__nv_bfloat16 *)Y, scale, (const uint16_t *)signs, early ? 1 : 0);
    });
}

// Few tokens: blocks for each, which read its A through L2 (3 TB/s or so, whatever the tokens' order); from 32 MB of such
// reads on the tile kernel, whose time goes by the adapters of a tile.  Whole calls at M = 1024, rows / tiles, us: K = 4096,
// rank 16, 128 tokens (16 MB) of one adapter 22.0 / 21.5, of eight 22.0 / 23.7; 256 tokens (32 MB) 26.3 / 25.6, 26.8 / 27.8;
// 512 (64 MB) 42 / 37, 43 / 38; 1024 (128 MB) 42 / 29, 42 / 30; rank 64, 64 tokens (32 MB) 22.5 / 20.9, 22.7 / 24.9; K = 1024,
// rank 64, 256 tokens (32 MB) 23.2 / 22.9, 23.3 / 24.7, 1024 (128 MB) 43 / 24; K = 8192, rank 16, 128 tokens (32 MB) 26.5 /
// 26.4, 26.5 / 31.4.  With 64 adapters in mixed order the rows stay ahead by a quarter beyond (1024 tokens 63 / 75), which
// the host cannot see.
static bool shrink_by_rows(int tokens, int K, int rank) { return (size_t)tokens * rank * K * 2 <= (size_t)32 << 20; }

static int launch_shrink_tiles(const void *X, const void *A, const int *index, const float *scaling, __nv_bfloat16 *S, int tokens, int K,
                               int adapters, int rank, cudaStream_t st)
{
    CUtensorMap tx, ta;
    int rc = encode_tmap_bf16_stack(&tx, X, 1, (uint64_t)tokens, (uint64_t)K, 256);
    if (rc) return rc;
    rc = encode_tmap_bf16_stack(&ta, A, (uint64_t)adapters, (uint64_t)rank, (uint64_t)K, (uint32_t)rank);
    if (rc) return rc;
    rc = ensure_dyn_smem((const void *)lora_shrink_tile_kernel, kShrinkSmem);
    if (rc) return rc;
    // K over a cluster of up to eight CTAs while all of them find an SM at once, then the passes over the adapters of a
    // tile over blockIdx.y the same way
    const int ntiles = (tokens + 255) / 256, per_pass = 128 / rank * 2;
    int split = 1;
    while (split < 8 && split * 2 <= K / 64 && ntiles * split * 2 <= sm_count()) split *= 2;
    const int most = adapters < 256 ? adapters : 256, passes = (most + per_pass - 1) / per_pass;
    int ways = sm_count() / (ntiles * split);
    ways = ways < 1 ? 1 : (ways > passes ? passes : ways);
    return launch_pdl_cluster(lora_shrink_tile_kernel, (unsigned)split, dim3((unsigned)(ntiles * split), (unsigned)ways),
                              dim3(kShrinkThreads), (size_t)kShrinkSmem, st, tx, ta, index, scaling, S, tokens, adapters, rank, K / 64,
                              split, status_word_ptr());
}

static int launch_front(const void *X, bool token_major, const void *A, const int *index, const float *scaling, __nv_bfloat16 *Xt, float *S,
                        int columns, int N, float scale, int adapters, int rank, cudaStream_t st)
{
    return with_logk<8>(ilog2((uint32_t)N), [&](auto logk) {
        constexpr int LOGK = decltype(logk)::value < 14 ? decltype(logk)::value : 13;   // the streaming GEMV ends at 8192
        if (token_major || columns == 1) {
            const int rows = shrink_rows_of_block(columns, rank), smem = N * 4;
            int rc = ensure_dyn_smem((const void *)lora_front_kernel<false, LOGK>, smem);
            if (rc) return rc;
            return launch_pdl(lora_front_kernel<false, LOGK>, dim3((unsigned)(columns * (1 + (rank + rows - 1) / rows))), dim3(256),
                              (size_t)smem, st, (const __nv_bfloat16 *)X, (const __nv_bfloat16 *)A, index, scaling, Xt, S, columns, scale,
                              adapters, rank, rows);
        }
        int rows = 1;   // rows of A at a time, of the seventh that a CTA has
        while (rows < 8 && rows < (rank + 6) / 7) rows *= 2;
        const int smem = N * 2 + N * 4;
        int rc = ensure_dyn_smem((const void *)lora_front_kernel<true, LOGK>, smem);
        if (rc) return rc;
        return launch_pdl_cluster(lora_front_kernel<true, LOGK>, 8, dim3((unsigned)columns * 8), dim3(256), (size_t)smem, st,
                                  (const __nv_bfloat16 *)X, (const __nv_bfloat16 *)A, index, scaling, Xt, S, columns, scale, adapters, rank,
                                  rows);
    });
}

static size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

// A decoding batch of B columns (or, token_major, tokens) of N elements in two launches: H(X) and S, then the streaming GEMV.
static int lora_stream(const void *W, const void *X, bool token_major, void *Y, size_t y_row, size_t y_column, const void *A, const void *Bm,
                       const int *index, const float *scaling, int M, int N, int B, int adapters, int rank, int out_dtype, float scale,
                       void *workspace, cudaStream_t st)
{
    __nv_bfloat16 *Xt = (__nv_bfloat16 *)workspace;
    float *S = (float *)((unsigned char *)workspace + up256((size_t)N * B * 2));
    const int rc = launch_front(X, token_major, A, index, scaling, Xt, S, B, N, scale, adapters, rank, st);
    if (rc) return rc;
    return launch_gemv_adapt(W, Xt, Y, M, N, B, out_dtype, GemvAdapt{Bm, S, index, adapters, rank, y_row, y_column}, st);
}

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
    // H(X); S in bf16 and the tables, or (few tokens) S in fp32
    const size_t s16 = up256((size_t)N * lora_pitch(rank) * 2) + up256(((size_t)N + 255) / 256 * kLoraTileInts * sizeof(int));
    const size_t s32 = gemv_adapt_shape(K, N) ? up256((size_t)N * rank * sizeof(float)) : 0;
    return b200ht_fused_gemm_workspace_bytes(M, N, K, B200HT_BF16) + (s16 > s32 ? s16 : s32);
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
    // as few tokens as the streaming GEMV serves with one pass over W; us, so / by what follows: 16 tokens at 4096 x 4096
    // 15 / 23, 4096 x 28672 72 / 101; 8 at 8192 x 1024 14.0 / 15.7, 8192 x 28672 105 / 124; 24 at 2048 x 4096 12.6 / 17.6; 32 at
    // 1024 x 4096 16.1 / 16.0, 512 x 512 13.7 / 14.7; one token 7.5 / 11.7 to 77 / 198
    if (!signs && gemv_adapt_shape(K, N)) {
        const bool mn = out_layout == B200HT_OUT_MN;
        return lora_stream(W, X, true, C, mn ? (size_t)N : 1, mn ? 1 : (size_t)M, A, B, index, scaling, M, K, N, adapters, rank, out_dtype,
                           scale, workspace, st);
    }
    unsigned char *ws = (unsigned char *)workspace + b200ht_fused_gemm_workspace_bytes(M, N, K, B200HT_BF16);
    __nv_bfloat16 *S = (__nv_bfloat16 *)ws;
    int *tiles = (int *)(ws + up256((size_t)N * lora_pitch(rank) * 2));
    const unsigned ntiles = (unsigned)((N + 255L) / 256);
    rc = launch_pdl(lora_plan_kernel, dim3(ntiles), dim3(256), 0, st, index, N, adapters, tiles);
    if (rc) return rc;
    rc = shrink_by_rows(N, K, rank) ? launch_shrink_rows(X, A, index, scaling, S, N, K, adapters, rank, 1, true, st)
                                    : launch_shrink_tiles(X, A, index, scaling, S, N, K, adapters, rank, st);
    if (rc) return rc;
    const LoraGemm lora{B, S, tiles, index, adapters, M, rank, 0};
    return fused_gemm_bf16_lora(X, W, C, M, N, K, out_dtype, out_layout, scale, signs, workspace, st, lora);
}

extern "C" size_t b200ht_lora_gemv_workspace_bytes(int M, int N, int B, int rank)
{
    using namespace b200ht;
    if (M <= 0 || N <= 0 || B <= 0 || rank <= 0) return 0;
    const size_t base = gemv_adapt_shape(N, B) ? (size_t)N * B * 2 : (size_t)M * B * sizeof(float);   // H(X), or W . H(X)
    return up256(base) + up256((size_t)B * rank * sizeof(float));
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
    if (!workspace || workspace_bytes < b200ht_lora_gemv_workspace_bytes(M, N, B, rank)) return B200HT_ERR_WORKSPACE;
    if ((uintptr_t)workspace & 255u) return B200HT_ERR_ALIGN;
    rc = check_device();
    if (rc) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    if (gemv_adapt_shape(N, B))
        return lora_stream(W, X, false, Y, (size_t)B, 1, A, Bm, index, scaling, M, N, B, adapters, rank, out_dtype, scale, workspace, st);
    float *base = (float *)workspace, *S = (float *)((unsigned char *)workspace + up256((size_t)M * B * sizeof(float)));
    rc = launch_shrink_rows(X, A, index, scaling, S, B, N, adapters, rank, B, false, st);
    if (rc) return rc;
    rc = b200ht_fused_gemv(W, X, base, M, N, B, B200HT_BF16, B200HT_F32, scale, stream);
    if (rc) return rc;
    int lanes = 1;
    while (lanes * 8 < rank) lanes *= 2;
    return launch_pdl(lora_expand_kernel, dim3((unsigned)((M + kExpandRows - 1) / kExpandRows)), dim3(256),
                      (size_t)kExpandRows * B * sizeof(float), st, (const float *)base, (const __nv_bfloat16 *)Bm, (const float *)S,
                      index, Y, M, B, adapters, rank, lanes, out_dtype);
}
