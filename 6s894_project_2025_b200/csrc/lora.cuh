// Low-rank adapters beside W . H(X): what the contraction (gemm_tcgen05.cu) and the adapters' own kernels (lora.cu) share.
#pragma once
#include "common.cuh"

namespace b200ht {

constexpr int kLoraMaxRank = 128;
// Table of one 256-token tile, made by lora_plan_kernel: the number of adapters among its tokens and their numbers, in
// the order of first appearance; 256 bits: tokens with an adapter; 256 bits for each adapter of the list: its tokens.
constexpr int kLoraValidOffset = 257, kLoraOwnOffset = kLoraValidOffset + 8, kLoraTileInts = kLoraOwnOffset + 256 * 8;

// Elements from one token's low-rank vector to the next: whole lines of 128 bytes, so that the copies of a tile by all CTAs
// at once spread over the L2 (256 tokens of rank 16 side by side are 64 lines; 128 CTAs fetching them for 16 adapters each
// took 15 us longer than with a line a token).
constexpr int lora_pitch(int rank) { return (rank + 63) & ~63; }

// The adapters of one contraction, as its launcher takes them.
struct LoraGemm {
    const void *B;       // [adapters][M][rank] bf16
    const void *S;       // [tokens][lora_pitch(rank)] bf16, rank of each used: scaling * A x of each token's adapter, 0 without one
    const int *tiles;    // kLoraTileInts per 256-token tile
    const int *index;    // adapter of each token
    int adapters, M, rank;
    int row;             // row of B that belongs to the first row of C

    // The same from row `r` and token `t` (a multiple of 256) on.
    LoraGemm at(long r, long t) const
    {
        LoraGemm o = *this;
        o.row += (int)r;
        o.S = (const unsigned char *)S + (size_t)t * lora_pitch(rank) * 2;
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
    size_t y_row, y_column;   // strides of the result in elements: one row of W, one column of X
};

}  // namespace b200ht
