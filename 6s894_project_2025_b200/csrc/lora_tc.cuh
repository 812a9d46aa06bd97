// Device pieces of the contractions with adapters (gemm_tcgen05.cu, lora_gemm.cu) and of the kernels around them.
#pragma once
#include "lora.cuh"
#include "tc_common.cuh"

namespace b200ht {

constexpr int kLoraTile = 256;   // tokens of a tile of the tables

// The adapters as operands of the tensor cores.
struct LoraOperands {
    CUtensorMap tmB;     // [adapter][M][rank]
    CUtensorMap tmS;     // [token][rank]
    const int *tiles;    // kLoraTileInts a 256-token tile: number of its adapters, their numbers, ...
    int rank;
    int row;             // row of B of this launch's first row of C
    // the operands in memory, for lora_unspoilt
    const __nv_bfloat16 *W, *Y, *B, *S;
    const int *index;
    int K, M, N, rows_b, adapters;   // of this launch; rows_b: rows of an adapter's B
};

// Host: [d2][d1][d0] bf16, rows of d0 contiguous values `pitch` apart (a multiple of 8; 0: d0), boxes of 1 x box1 x 64 with
// 128-byte swizzle; a box that reaches beyond d0 or d1 is filled with zeros.
int encode_tmap_bf16_stack(CUtensorMap *map, const void *base, uint64_t d2, uint64_t d1, uint64_t d0, uint32_t box1,
                           uint64_t pitch = 0);
int lora_operands(LoraOperands *o, const LoraGemm &lora, const void *W, const void *Y, int M, int N, int K, int rows, int box);

// An adapter's B is multiplied with zeros for the other tokens of a group of 16, and an infinity or NaN in it makes NaN of
// their results.  The epilogues therefore look for values that are not finite (a multiplication by zero a value; calls of
// sound adapters take as long as without, 0.97 .. 1.03 times at 16384 x 8192 x 28672 under the power cap, 0.99 .. 1.01 at
// 64 .. 4096 tokens) and ask here for C[m, t]: `v` itself, unless row m of another adapter in token t's group holds such a
// value; then the sums of W . H(X) and of the token's own adapter, again, by one thread in fp32.  That is slow (2048 tokens
// of 16 adapters in mixed order, one of them NaN throughout, 8192 x 4096: 36 .. 57 ms for 0.2; 25 ms a tile, far within
// the time limit of the other warps' waits), but no token's result depends on another's adapter.
static __device__ __noinline__ float lora_unspoilt(const LoraOperands &o, int m, int t, float v)
{
    const auto not_finite = [](uint32_t two) { return (two & 0x7f80u) == 0x7f80u || (two & 0x7f800000u) == 0x7f800000u; };
    const int own = o.index[t], from = t & ~15, to = from + 16 < o.N ? from + 16 : o.N;
    bool spoilt = false;
    for (int u = from, last = own; u < to && !spoilt; ++u) {
        const int a = o.index[u];
        if (a == own || a == last || (unsigned)a >= (unsigned)o.adapters) continue;
        last = a;
        const uint4 *b = (const uint4 *)(o.B + ((size_t)a * o.rows_b + o.row + m) * o.rank);
        for (int i = 0; i < o.rank / 8; ++i) {
            const uint4 p = b[i];
            spoilt |= not_finite(p.x) || not_finite(p.y) || not_finite(p.z) || not_finite(p.w);
        }
    }
    if (!spoilt) return v;
    float2 s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = make_float2(0.f, 0.f);
    const auto add = [&](const uint4 &p, const uint4 &q) {
        const uint32_t pw[4] = {p.x, p.y, p.z, p.w}, qw[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 a = unpack2<B200HT_BF16>(pw[i]), b = unpack2<B200HT_BF16>(qw[i]);
            s[i].x = fmaf(a.x, b.x, s[i].x);
            s[i].y = fmaf(a.y, b.y, s[i].y);
        }
    };
    const uint4 *w = (const uint4 *)(o.W + (size_t)m * o.K), *y = (const uint4 *)(o.Y + (size_t)t * o.K);
#pragma unroll 8
    for (int k = 0; k < o.K / 8; ++k) add(w[k], y[k]);
    if ((unsigned)own < (unsigned)o.adapters) {
        const uint4 *b = (const uint4 *)(o.B + ((size_t)own * o.rows_b + o.row + m) * o.rank);
        const uint4 *x = (const uint4 *)(o.S + (size_t)t * lora_pitch(o.rank));
        for (int i = 0; i < o.rank / 8; ++i) add(b[i], x[i]);
    }
    return ((s[0].x + s[0].y) + (s[1].x + s[1].y)) + ((s[2].x + s[2].y) + (s[3].x + s[3].y));
}

__device__ __forceinline__ bool all_finite(const uint32_t (&r)[32])   // fp32 bits
{
    float z[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 32; ++j) z[j & 3] = fmaf(__uint_as_float(r[j]), 0.f, z[j & 3]);   // NaN from the first that is not
    return (z[0] + z[1]) + (z[2] + z[3]) == 0.f;
}

// The same for the 32 columns of the accumulator from `taddr` on (tokens n .. n + 31), one row m of C a lane.  By one warp.
static __device__ __noinline__ void lora_unspoil_columns(const LoraOperands &o, uint32_t taddr, int m, int n)
{
#pragma unroll 1
    for (int j = 0; j < 32; ++j) {
        uint32_t v;
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n" : "=r"(v) : "r"(taddr + j) : "memory");
        tmem_ld_wait();
        if (m < o.M && n + j < o.N && isnan(__uint_as_float(v))) v = __float_as_uint(lora_unspoilt(o, m, n + j, __uint_as_float(v)));
        __syncwarp();
        asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};\n" ::"r"(taddr + j), "r"(v) : "memory");
    }
    asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
}

// The same for 32 results already in bf16, `step` elements apart in shared memory, one row m a lane.
static __device__ __noinline__ void lora_unspoil_staged(const LoraOperands &o, __nv_bfloat16 *at, int step, int m, int n)
{
#pragma unroll 1
    for (int j = 0; j < 32; ++j) {
        const float v = __bfloat162float(at[j * step]);
        if (m < o.M && n + j < o.N && isnan(v)) at[j * step] = __float2bfloat16_rn(lora_unspoilt(o, m, n + j, v));
    }
}

// One warp's walk over entries first, first + step, ... of a tile's list: lane w < 8 gets word w of the tokens with an
// adapter, and of those of the entry's.  Four entries a load, the next four under way.
struct LoraTileWalk {
    const int *tile;
    int count, at, step;      // entries of the list; the next one to hand out
    uint32_t valid, now, ahead;

    __device__ __forceinline__ uint32_t fetch(int entry, int lane) const
    {
        entry += (lane >> 3) * step;
        return entry < count ? (uint32_t)__ldcg(tile + kLoraOwnOffset + entry * 8 + (lane & 7)) : 0u;
    }
    __device__ __forceinline__ void start(const int *t, int first, int by, int lane)
    {
        tile = t;
        at = first;
        step = by;
        valid = lane < 8 ? (uint32_t)__ldcg(t + kLoraValidOffset + lane) : 0u;
        count = __ldcg(t);
        // before the count is known: all 256 entries have their place in the table
        now = (uint32_t)__ldcg(t + kLoraOwnOffset + min(first + (lane >> 3) * by, 255) * 8 + (lane & 7));
        ahead = 0;
        taken = 0;
    }
    __device__ __forceinline__ bool more() const { return at < count; }
    __device__ __forceinline__ uint32_t next(int lane)   // by the whole warp
    {
        if (taken == 0) ahead = fetch(at + 4 * step, lane);
        const uint32_t word = __shfl_sync(0xffffffffu, now, taken * 8 + (lane & 7));
        at += step;
        if (++taken == 4) {
            taken = 0;
            now = ahead;
        }
        return lane < 8 ? word : 0u;
    }
    int taken;                // of the four
};

// Bit i of the low eight at bit 2 i.
__device__ __forceinline__ uint32_t spread_bits(uint32_t x)
{
    x = (x | (x << 4)) & 0x0f0fu;
    x = (x | (x << 2)) & 0x3333u;
    return (x | (x << 1)) & 0x5555u;
}

// Groups of 16 tokens (bit g: tokens 16 g .. 16 g + 15 of the tile of 128-byte rows at `rows`) that have a token of `own`.
// In these groups the rows of tokens with another adapter are set to zero; those of tokens without one are zero already.
// By one warp.  Short code rather than unrolled: it runs a few times a tile and costs most by being fetched.
__device__ __forceinline__ uint32_t lora_groups(uint32_t rows, uint32_t own, uint32_t valid, int lane)
{
    const uint32_t other = valid & ~own;
    const bool lo = own & 0xffffu, hi = own >> 16;
    const uint32_t groups = spread_bits(__ballot_sync(0xffffffffu, lo)) | (spread_bits(__ballot_sync(0xffffffffu, hi)) << 1);
    uint32_t mixed = spread_bits(__ballot_sync(0xffffffffu, lo && (other & 0xffffu))) |
                     (spread_bits(__ballot_sync(0xffffffffu, hi && (other >> 16))) << 1);
    if (mixed) {
#pragma unroll 1
        for (; mixed; mixed &= mixed - 1) {
            const int g = __ffs(mixed) - 1;
            const uint32_t bits = __shfl_sync(0xffffffffu, other, g >> 1) >> (16 * (g & 1));
#pragma unroll
            for (int r = 0; r < 16; r += 4) {   // four rows an instruction
                const int row = r + (lane >> 3);
                if ((bits >> row) & 1u)
                    asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};\n" ::"r"(rows + (uint32_t)((g * 16 + row) * 128 + (lane & 7) * 16)),
                                 "r"(0)
                                 : "memory");
            }
        }
        fence_proxy_async();
        __syncwarp();
    }
    return groups;
}

// D[:, tokens of `groups`] += B . S^T for 128 rows of B at `b` and the tokens at `s`: one instruction for each stretch of
// neighbouring groups and 16 of the `left` (at most 64 used) columns of the rank.  One thread.
__device__ __forceinline__ void lora_mma_groups(uint32_t d_tmem, uint32_t b, uint32_t s, uint32_t groups, int left)
{
    const int ksteps = left >= 64 ? 4 : (left + 15) / 16;
    const uint64_t bdesc = umma_desc_k_sw128(b);
    while (groups) {
        const int g0 = __ffs(groups) - 1, n = __ffs(~(groups >> g0)) - 1;
        groups &= ~(((1u << n) - 1) << g0);
        const uint64_t sdesc = umma_desc_k_sw128(s + g0 * 2048);
        const uint32_t idesc = umma_idesc_bf16(128, 16 * n);
        for (int k = 0; k < ksteps; ++k) umma_bf16_ss(d_tmem + 16 * g0, bdesc + 2 * k, sdesc + 2 * k, idesc, 1u);
    }
}

// All threads of all CTAs of the cluster.
__device__ __forceinline__ void cluster_sync_all()
{
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}

// launch_pdl with clusters of `cluster` CTAs along x.
template <typename... KArgs, typename... Args>
inline int launch_pdl_cluster(void (*kernel)(KArgs...), unsigned cluster, dim3 grid, dim3 block, size_t smem, cudaStream_t st, Args... args)
{
    note_launch();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return (int)cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

}  // namespace b200ht
