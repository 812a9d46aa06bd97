// Low-rank adapters beside W . H(X): what the contraction (gemm_tcgen05.cu) and the adapters' own kernels (lora.cu) share.
#pragma once
#include "common.cuh"

namespace b200ht {

constexpr int kLoraMaxRank = 128;
// Table of one 256-token tile, made by lora_plan_kernel: the number of adapters among its tokens and their numbers, then
// the same for each of its 128-token halves, each list in the order of first appearance.
constexpr int kLoraHalfOffset = 257, kLoraHalfInts = 129;
constexpr int kLoraTileInts = 516;   // 1 + 256 + 2 * (1 + 128), to a multiple of four

// The adapters of one contraction, as its launcher takes them.
struct LoraGemm {
    const void *B;       // [adapters][M][rank] bf16
    const void *S;       // [tokens][rank] bf16: scaling * A x of each token's adapter, 0 without one
    const int *tiles;    // kLoraTileInts per 256-token tile
    const int *index;    // adapter of each token
    int adapters, M, rank;
    int row;             // row of B that belongs to the first row of C

    // The same from row `r` and token `t` (a multiple of 256) on.
    LoraGemm at(long r, long t) const
    {
        LoraGemm o = *this;
        o.row += (int)r;
        o.S = (const unsigned char *)S + (size_t)t * rank * 2;
        o.tiles = tiles + (size_t)(t / 256) * kLoraTileInts;
        o.index = index + t;
        return o;
    }
};

// The adapters of a decoding batch, as the streaming GEMV takes them.
struct GemvAdapt {
    const void *B;       // [adapters][M][rank] bf16
    const float *S;      // [columns][rank]
    const int *index;    // adapter of each column
    int adapters, rank;
};

}  // namespace b200ht
