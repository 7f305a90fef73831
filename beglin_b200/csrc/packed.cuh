// A cache in 4 bits: how a page holds keys and values, and how they are read back.
//
// For each kv head a page [page_size positions] is a run of tiles of 16 positions, each
//     keys' codes | values' codes | (step, lowest) pairs of every position
// and a position's value for feature f is lowest + step u, u its code in 0 .. 15 and (step, lowest) the pair, in bfloat16, of f's group of 64
// features of that position's key (or value).  Behind the tiles may stand the smallest and the largest value of every feature of the page's keys.
// 4.5 bits a value: 2,304 bytes a tile of heads of 128 features, and any run of tiles is one run of bytes, so that one bulk copy brings it.
//
// The codes lie as the m16n8k16 product takes its left operand, so that a lane loads its fragment as it is:
//   keys    position p at p * HD/2; in it, quarter t (lane % 4), group, two words of 8 features: features 64 group + 16 t + 8 w .. + 7.  A word's nibble
//           i < 4 is its feature 2 i, nibble 4 + i its feature 2 i + 1: shifted by 4 i and masked with 0x000f000f it is a pair of neighbours.
//   values  lane 4 g + t holds, of positions 2t, 2t+1, 2t+8, 2t+9, the features 64 group + 8 g .. + 7 as one word each (nibble i: feature i).  Heads of 64:
//           16 bytes a lane, one word a position; heads of 128: two planes of 16 bytes a lane, a plane two positions of two words (the groups).
#pragma once
#include "ptx.cuh"

namespace bg {

constexpr int PK_TILE = 16, PK_GROUP = 64;
constexpr int PK_WIDE = 64;                // positions of a page written out in half precision

// What is written out with the pages of a kv head of a request: its keys are written times 2^-keys and its values times 2^-values; bit g of `marked`: some of its
// values' g-th groups are no numbers. Those are written as noughts and marked, a bit a position of a page: a product would carry them to the rows
// that do not see them, whose weight for them is nought.
// `base`: its page i (of PK_WIDE positions) is page base + i of what is written out.
struct __align__(16) PkWritten { int keys, values, marked, base; };

// Pages that `rows` rows need whose last position lies below `end`: the requests' lie one behind the other, each with room for what it reads, not for the longest.
__host__ __device__ inline int packed_room(int rows, int end, int window) {
    const int whole = end > 0 ? (end - 1) / PK_WIDE + 1 : 1;
    if (window <= 0) return whole;
    const long long span = ((long long)rows + window - 2 + PK_WIDE - 1) / PK_WIDE + 1;          // (rows + window - 1 positions, wherever they begin in a page)
    return span < whole ? (int)span : whole;
}

template <int HD>
struct Packed {
    static constexpr int GROUPS = HD / PK_GROUP;
    static constexpr int CODES = PK_TILE * HD / 2;              // bytes of a tile's keys, and of its values
    static constexpr int PAIRS = 2 * CODES;                     // where the (step, lowest) pairs begin
    static constexpr int TILE = PAIRS + PK_TILE * 2 * GROUPS * 4;

    // Where the word of 8 features from `f` (a multiple of 8) of the tile's position p begins.
    __host__ __device__ static constexpr int key_word(int p, int f) {
        return p * (HD / 2) + ((f % PK_GROUP) / 16 * GROUPS + f / PK_GROUP) * 8 + (f % 16) / 8 * 4;
    }
    __host__ __device__ static constexpr int value_word(int p, int f) {
        const int lane = (f % PK_GROUP) / 8 * 4 + p % 8 / 2;
        return CODES + (GROUPS == 2 ? p / 8 * 512 + lane * 16 + p % 2 * 8 + f / PK_GROUP * 4 : lane * 16 + (p / 8 * 2 + p % 2) * 4);
    }
    __host__ __device__ static constexpr int pair_word(int p, int value, int group) { return PAIRS + (p * 2 * GROUPS + value * GROUPS + group) * 4; }
};

__host__ __device__ inline long long packed_tile_bytes(int hd) { return hd == 64 ? Packed<64>::TILE : Packed<128>::TILE; }

__device__ __forceinline__ float pair_step(unsigned pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float pair_lowest(unsigned pair) { return __uint_as_float(pair & 0xffff0000u); }
__device__ __forceinline__ bool pair_finite(unsigned pair) { return fabsf(fmaf(15.0f, pair_step(pair), pair_lowest(pair))) < INFINITY; }

// The power of two (times 2^14) of the largest of some numbers: less that, they lie below 2^15, where half precision holds them whatever their scale is. 2^-this
// is a normal number too.
__device__ __forceinline__ int half_shift(float largest) { return min(113, max(-126, (int)(__float_as_uint(largest) >> 23) - 127 - 14)); }

// The 8 values of a word of codes (KEY: a key's order of nibbles).
template <bool KEY>
__device__ __forceinline__ void packed_values(unsigned word, unsigned pair, float (&v)[8]) {
    const float step = pair_step(pair), lowest = pair_lowest(pair);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int nib = KEY ? e / 2 + 4 * (e % 2) : e;
        v[e] = fmaf(step, (float)((word >> (4 * nib)) & 15u), lowest);        // (the product is exact: 8 by 4 bits)
    }
}

}  // namespace bg
