// C = W . Y + B S for few tokens: the contraction of gemm_tcgen05.cu with adapters, where its tiles would leave most SMs
// without work (a decoding batch of 64 at M = 4096 has 32).  The CTAs of a cluster share a tile: each takes a part of K
// and every split-th adapter, and at the end adds up 1 / split of the tile's tokens from all of them through distributed
// shared memory, in the order of the ranks.
//
//   warp 0      TMA producer: W (128 x 64) and Y (`box` tokens x 64) a stage, then B (128 x 64) and S of each adapter.
//               W's first stages are requested before the kernel in front (the transform) has finished: the chain starts
//               after all earlier work (lora_plan_kernel), so W is complete.
//   warp 1      tcgen05.mma (M = 128, N = box, K = 16); masks S as gemm_tcgen05.cu does
//   warps 2..5  the accumulator into shared memory, over the used stages, one row of W a lane
// Bound: the bytes of W, and the chain of four launches (plan, S, H(X), this), each of which waits for its latencies; a
// CTA's time goes by its K steps, hence the split over K.  64 tokens of 16 adapters (rank 16) at 4096 x 4096: 24 us with
// everything in front (6 at the copy bandwidth), 50 by the tiles of gemm_tcgen05.cu.  Every wait is time-limited; a CTA whose wait ran out keeps step with its cluster and leaves
// B200HT_ERR_TIMEOUT in the status word.
#include "lora_tc.cuh"

namespace b200ht {

constexpr int kSplitThreads = 192, kSplitRing = 192 * 1024;
constexpr int kSplitPitch = 132;   // floats of a token's row of partial sums: 128 rows of W, a multiple of 16 bytes
static_assert(256 * kSplitPitch * 4 <= kSplitRing, "the partial sums lie over the ring");

template <int OUT_DT, int LAYOUT>
__global__ void __launch_bounds__(kSplitThreads, 1)
lora_gemm_split_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmY,
                       const __grid_constant__ LoraOperands lora, void *C, int M, int N, int kblocks, int box, int stages, int split,
                       int *status)
{
    extern __shared__ unsigned char smem_dyn[];
    const uint32_t base = (smem_u32(smem_dyn) + 1023u) & ~1023u;
    unsigned char *gen = smem_dyn + (base - smem_u32(smem_dyn));
    const int stage_bytes = 16384 + box * 128;
    const uint32_t bars = base + kSplitRing;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 64u + 8u * s; };   // at most eight stages
    const uint32_t done_bar = bars + 128u;
    uint32_t *tmem_slot = (uint32_t *)(gen + kSplitRing + 136);
    volatile int *abort_flag = (volatile int *)(tmem_slot + 1);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int part = blockIdx.x % split, m0 = blockIdx.x / split * 128, nb = blockIdx.y, n0 = nb * kLoraTile;

    if (tid == 0) {
        for (int s = 0; s < stages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(done_bar, 1);
        *abort_flag = 0;
        fence_barrier_init();
        tma_prefetch_desc(&tmW);
        tma_prefetch_desc(&tmY);
    }
    if (warp == 1) tmem_alloc(smem_u32(tmem_slot), (uint32_t)box);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();
    const int nk = kblocks / split, kb0 = part * nk;
    const int ahead = nk < stages ? nk : stages;
    if (warp == 0 && lane == 0)
        for (int i = 0; i < ahead; ++i) {
            mbar_expect_tx(full_bar(i), (uint32_t)stage_bytes);
            tma_load_2d(base + i * stage_bytes, &tmW, (kb0 + i) * 64, m0, full_bar(i));
        }
    __syncwarp();
    pdl_wait();

    bool ok = true;
    if (warp == 0) {
        if (lane == 0) {
            const int *tile = lora.tiles + (size_t)nb * kLoraTileInts;
            const int count = __ldcg(tile);
            int it = 0, queue[4];   // this CTA's next adapters
#pragma unroll
            for (int i = 0; i < 4; ++i) queue[i] = __ldcg(tile + 1 + part + i * split);   // entries up to 31: in the table
            for (; it < nk; ++it) {
                const int s = it % stages;
                const uint32_t sa = base + s * stage_bytes;
                if (it >= ahead) {
                    if (!mbar_wait(empty_bar(s), ((it / stages) & 1u) ^ 1u, abort_flag, status)) { ok = false; break; }
                    mbar_expect_tx(full_bar(s), (uint32_t)stage_bytes);
                    tma_load_2d(sa, &tmW, (kb0 + it) * 64, m0, full_bar(s));
                }
                tma_load_2d(sa + 16384, &tmY, (kb0 + it) * 64, n0, full_bar(s));
            }
            for (int i = part; i < count && ok; i += split) {
                const int adapter = queue[0];
                queue[0] = queue[1], queue[1] = queue[2], queue[2] = queue[3];
                if (i + 4 * split < count) queue[3] = __ldcg(tile + 1 + i + 4 * split);
                for (int r = 0; r < lora.rank; r += 64, ++it) {
                    const int s = it % stages;
                    if (!mbar_wait(empty_bar(s), ((it / stages) & 1u) ^ 1u, abort_flag, status)) { ok = false; break; }
                    mbar_expect_tx(full_bar(s), (uint32_t)stage_bytes);
                    tma_load_3d(base + s * stage_bytes, &lora.tmB, r, lora.row + m0, adapter, full_bar(s));
                    tma_load_3d(base + s * stage_bytes + 16384, &lora.tmS, r, n0, 0, full_bar(s));
                }
            }
            if (!ok) {   // copies on their way still land in this CTA's shared memory: give them time
                const int pending = it < stages ? it : stages;
                for (int j = 1; j <= pending; ++j) {
                    const uint64_t ns = global_ns();
                    while (!mbar_test(full_bar((it - j) % stages), ((it - j) / stages) & 1u) && global_ns() - ns < 100000000ull) {}
                }
            }
        }
    } else if (warp == 1) {
        LoraTileWalk walk;
        walk.start(lora.tiles + (size_t)nb * kLoraTileInts, part, split, lane);
        const uint32_t idesc = umma_idesc_bf16(128, box);
        int it = 0;
        if (lane == 0)
            for (; it < nk; ++it) {
                const int s = it % stages;
                if (!mbar_wait(full_bar(s), (it / stages) & 1u, abort_flag, status)) { ok = false; break; }
                tc_fence_after();
                const uint32_t sa = base + s * stage_bytes;
                const uint64_t adesc = umma_desc_k_sw128(sa), bdesc = umma_desc_k_sw128(sa + 16384);
#pragma unroll
                for (int k = 0; k < 4; ++k) umma_bf16_ss(tmem, adesc + 2 * k, bdesc + 2 * k, idesc, (it | k) ? 1u : 0u);
                umma_commit(empty_bar(s));
            }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        it = nk;
        while (walk.more() && ok) {
            const uint32_t own = walk.next(lane);
            for (int r = 0; r < lora.rank; r += 64, ++it) {
                const int s = it % stages;
                ok = __all_sync(0xffffffffu, mbar_wait(full_bar(s), (it / stages) & 1u, abort_flag, status));
                if (!ok) break;
                const uint32_t sa = base + s * stage_bytes;
                const uint32_t groups = lora_groups(sa + 16384, own, walk.valid, lane);
                if (lane == 0) {
                    tc_fence_after();
                    lora_mma_groups(tmem, sa, sa + 16384, groups, lora.rank - r);
                    umma_commit(empty_bar(s));
                }
                __syncwarp();
            }
        }
        if (ok && lane == 0) umma_commit(done_bar);
    }
    __syncwarp();
    // all MMAs done: the accumulator is complete, the ring free
    ok = mbar_wait(done_bar, 0u, abort_flag, status);
    ok = __syncthreads_and(ok);
    float *sums = (float *)gen;   // [token][kSplitPitch]
    const int tokens = N - n0 < box ? N - n0 : box;
    if (ok && warp >= 2) {
        tc_fence_after();
        const int q = warp & 3, row = q * 32 + lane;
        for (int c = 0; c < tokens; c += 32) {   // box is a multiple of 32: columns behind the last token are read, not kept
            uint32_t v[32];
            tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + c, v);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (c + i < tokens) sums[(c + i) * kSplitPitch + row] = __uint_as_float(v[i]);
        }
        tc_fence_before();
    }
    cluster_sync_all();
    const int per = (tokens + split - 1) / split, t1 = (part + 1) * per < tokens ? (part + 1) * per : tokens;
    for (int t = part * per + warp; t < t1 && ok; t += kSplitThreads / 32) {
        float4 v[8], sum = make_float4(0.f, 0.f, 0.f, 0.f);
        const uint32_t at = base + (uint32_t)((t * kSplitPitch + 4 * lane) * 4);
#pragma unroll
        for (int p = 0; p < 8; ++p)
            if (p < split) {
                uint32_t there;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(there) : "r"(at), "r"(p));
                asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];\n"
                             : "=f"(v[p].x), "=f"(v[p].y), "=f"(v[p].z), "=f"(v[p].w)
                             : "r"(there)
                             : "memory");
            }
#pragma unroll
        for (int p = 0; p < 8; ++p)
            if (p < split) sum = make_float4(sum.x + v[p].x, sum.y + v[p].y, sum.z + v[p].z, sum.w + v[p].w);
        const int m = m0 + 4 * lane;
        float f[4] = {sum.x, sum.y, sum.z, sum.w};
        if (isnan(f[0]) || isnan(f[1]) || isnan(f[2]) || isnan(f[3])) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (m + e < M && isnan(f[e])) f[e] = lora_unspoilt(lora, m + e, n0 + t, f[e]);
            sum = make_float4(f[0], f[1], f[2], f[3]);
        }
        if (LAYOUT == B200HT_OUT_NM && (M & 3) == 0) {
            const size_t i = (size_t)(n0 + t) * M + m;
            if (m < M) {
                if constexpr (OUT_DT == B200HT_F32) *(float4 *)((float *)C + i) = sum;
                else *(uint2 *)((__nv_bfloat16 *)C + i) = make_uint2(pack2<B200HT_BF16>(f[0], f[1]), pack2<B200HT_BF16>(f[2], f[3]));
            }
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (m + e < M) {
                    const size_t i = LAYOUT == B200HT_OUT_NM ? (size_t)(n0 + t) * M + m + e : (size_t)(m + e) * N + n0 + t;
                    if constexpr (OUT_DT == B200HT_F32) ((float *)C)[i] = f[e];
                    else ((__nv_bfloat16 *)C)[i] = __float2bfloat16_rn(f[e]);
                }
        }
    }
    cluster_sync_all();   // nobody leaves while others read its sums
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, (uint32_t)box);
    }
}

// CTAs of a cluster for these sizes: doubled while all clusters find an SM a CTA at once and each CTA has two K steps of 64;
// 1 leaves the call to gemm_tcgen05.cu.
int lora_gemm_split(int M, int N, int K)
{
    const long tiles = (long)((M + 127) / 128) * ((N + kLoraTile - 1) / kLoraTile);
    int split = 1;
    while (split < 8 && tiles * split * 2 <= sm_count() && K / 64 >= 4 * split) split *= 2;
    return split;
}

template <int OUT_DT, int LAYOUT>
static int launch_split(const void *Y, const void *W, void *C, int M, int N, int K, int split, const LoraGemm &lora, cudaStream_t st)
{
    const int box = N <= 64 ? 64 : (N <= 128 ? 128 : 256), stages = kSplitRing / (16384 + box * 128);
    CUtensorMap tw, ty;
    int rc = encode_tmap_bf16_2d(&tw, W, (uint64_t)M, (uint64_t)K, 128);
    if (rc) return rc;
    rc = encode_tmap_bf16_2d(&ty, Y, (uint64_t)N, (uint64_t)K, (uint32_t)box);
    if (rc) return rc;
    LoraOperands o{};
    rc = lora_operands(&o, lora, W, Y, M, N, K, 128, box);
    if (rc) return rc;
    constexpr int smem = kSplitRing + 1024 + 256;
    rc = ensure_dyn_smem((const void *)lora_gemm_split_kernel<OUT_DT, LAYOUT>, smem);
    if (rc) return rc;
    return launch_pdl_cluster(lora_gemm_split_kernel<OUT_DT, LAYOUT>, (unsigned)split,
                              dim3((unsigned)((M + 127) / 128 * split), (unsigned)((N + kLoraTile - 1) / kLoraTile)), dim3(kSplitThreads),
                              (size_t)smem, st, tw, ty, o, C, M, N, K / 64, box, stages, split, status_word_ptr());
}

int launch_lora_gemm_split(const void *Y, const void *W, void *C, int M, int N, int K, int out_dtype, int out_layout, int split,
                           const LoraGemm &lora, cudaStream_t st)
{
    if (out_dtype == B200HT_F32)
        return out_layout == B200HT_OUT_MN ? launch_split<B200HT_F32, B200HT_OUT_MN>(Y, W, C, M, N, K, split, lora, st)
                                           : launch_split<B200HT_F32, B200HT_OUT_NM>(Y, W, C, M, N, K, split, lora, st);
    return out_layout == B200HT_OUT_MN ? launch_split<B200HT_BF16, B200HT_OUT_MN>(Y, W, C, M, N, K, split, lora, st)
                                       : launch_split<B200HT_BF16, B200HT_OUT_NM>(Y, W, C, M, N, K, split, lora, st);
}

}  // namespace b200ht
