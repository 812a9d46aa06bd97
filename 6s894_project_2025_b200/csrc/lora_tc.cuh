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
    const int *index;    // adapter of each token
    int adapters, rank;
    int row;             // row of B of this launch's first row of C
};

// Host: [d2][d1][d0] bf16, d0 contiguous (a multiple of 8), boxes of 1 x box1 x 64 with 128-byte swizzle; a box that
// reaches beyond d0 or d1 is filled with zeros.
int encode_tmap_bf16_stack(CUtensorMap *map, const void *base, uint64_t d2, uint64_t d1, uint64_t d0, uint32_t box1);
int lora_operands(LoraOperands *o, const LoraGemm &lora, int tokens, int rows, int box);

// Groups of 16 tokens (bit g: tokens 16 g .. 16 g + 15 of the tile of 128-byte rows at `tile`) that have a token of `adapter`.
// In these groups the rows (128 bytes each) of tokens with another adapter are set to zero; those of tokens without one
// are zero already.  `ids`: adapters of tokens lane, lane + 32, ... (negative: none).  One warp.
__device__ __forceinline__ uint32_t tc_adapter_groups(uint32_t tile, const int (&ids)[kLoraTile / 32], int adapter, int lane)
{
    uint32_t groups = 0, zeroed = 0;
#pragma unroll
    for (int i = 0; i < kLoraTile / 32; ++i) {
        const uint32_t own = __ballot_sync(0xffffffffu, ids[i] == adapter);
        const uint32_t other = __ballot_sync(0xffffffffu, ids[i] >= 0 && ids[i] != adapter);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const uint32_t bits = 0xffffu << (16 * h);
            if (!(own & bits)) continue;
            groups |= 1u << (2 * i + h);
            if (!(other & bits)) continue;
            zeroed = 1;
#pragma unroll
            for (int r = 0; r < 16; r += 4) {   // four rows an instruction
                const int row = 16 * h + r + (lane >> 3);
                if ((other >> row) & 1u)
                    asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};\n" ::"r"(tile + (uint32_t)((i * 32 + row) * 128 + (lane & 7) * 16)),
                                 "r"(0)
                                 : "memory");
            }
        }
    }
    if (zeroed) {
        fence_proxy_async();
        __syncwarp();
    }
    return groups;
}

// One warp's view of tile `nb`: adapters of tokens lane, lane + 32, ..., the list of the tile's adapters the same way.
// Returns their number.  (Numbers from `adapters` on are no adapters: the caller drops them once the loads have arrived.)
__device__ __forceinline__ int lora_tile_tables(const LoraOperands &o, int nb, int tokens, int lane, int (&ids)[kLoraTile / 32],
                                                int (&list)[kLoraTile / 32])
{
    const int *tile = o.tiles + (size_t)nb * kLoraTileInts;
#pragma unroll
    for (int i = 0; i < kLoraTile / 32; ++i) {
        const int n = nb * kLoraTile + i * 32 + lane;
        ids[i] = n < tokens ? __ldcg(o.index + n) : -1;
        list[i] = __ldcg(tile + 1 + i * 32 + lane);
    }
    return __ldcg(tile);
}
__device__ __forceinline__ int lora_list_entry(const int (&list)[kLoraTile / 32], int i)   // by the whole warp
{
    int entry = list[0];
#pragma unroll
    for (int j = 1; j < kLoraTile / 32; ++j) entry = i >> 5 == j ? list[j] : entry;
    return __shfl_sync(0xffffffffu, entry, i & 31);
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
