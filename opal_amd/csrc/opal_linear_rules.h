// Which kernel makes a matrix product of the score head (opal_linear.h): the rules, both sides of each as measured.  Host code without HIP, so that
// what a size reaches can be asked where there is no GPU.
#pragma once
#include <algorithm>
#include <cstdint>

#include "opal_hip.h"

namespace opal_head {

enum Product { FWD = 0, GIN = 1, GWT = 2 };

constexpr int STEP_BYTES = 128;          // of k per row and step of the tile kernels

inline int type_bytes(int type) { return type == OPAL_F32 ? 4 : 2; }

// Tiles by number: 0 = 64 x 64, 1 = 128 x 128, 2 = 256 x 256 (16-bit types on the aligned path only), 3 = few rows (no fixed height), 4 = 128 x 256
// (FWD, as 2), 5 = 32 x 32 over all rows (GWT).
constexpr int TILE_M[] = {64, 128, 256, 0, 128, 32}, TILE_N[] = {64, 128, 256, 0, 256, 32};

inline uint64_t tiles_of(uint64_t M, uint64_t N, int tile) { return ((M + TILE_M[tile] - 1) / TILE_M[tile]) * ((N + TILE_N[tile] - 1) / TILE_N[tile]); }

// Larger tiles read fewer bytes for the same sums, smaller ones leave fewer CUs idle and less of a tile outside the matrix (us; rows x N x K):
//   128 x 128 instead of 64 x 64, 16-bit types, sums of 512 on, from 1.5 tiles a CU on: 16384 x 1564 x 512 34.5 against 49.3, 100 000 x 128 x 1000 49
//   against 56; below it 4096 x 1564 x 512 (416) 14.4 against 15.1; shorter sums 100 000 x 200 x 200 24.4 against 21.8.  Not where it reaches a
//   quarter further: 100 000 x 150 x 1000 90 against 83, 100 000 x 64 x 512 26 against 20.  32-bit types, bound by the matrix pipe, never: 50 000 x
//   512 x 1564 694 against 674, 100 000 x 200 x 150 126 against 82.
// 16-bit types, aligned:
//   256 x 256 from one tile a CU on.  Input gradients where it does not reach a quarter further than 128 x 128: 32768 x 512 x 256 17.5 against 22.3, 100 000 x
//   600 x 64 35 against 44; but 100 000 x 356 x 1000 125 against 113.  Forward products, which have 128 x 256 tiles too, with more than
//   128 columns and sums of 1024 on (32768 x 512 x 1564 (256) 51 against 59; below it 16384 x 512 x 1564 (128) 38 against 32), or of 256 on from
//   four tiles a CU on: 250 000 x 355 x 256 (1954) 106 against 110, 100 000 x 1563 x 256 140 against 169; below it 100 000 x 512 x 512 (782) 76
//   against 70, 32768 x 1564 x 512 (896) 72 against 68.
//   128 x 256 (forward, more than 128 columns) from 3/4 of a tile a CU on: 250 000 x 355 x 128 66 against 82 with 256 x 256 and 104 with 128 x 128, 4096 x
//   1564 x 512 (224) 14.1 against 15.5; below it 4099 x 512 x 355 (66) 12.2 against 10.9, 16384 x 200 x 200 (128) 10.9 against 7.7.
// large: the last two may take it; whole: the first of them too.
inline uint64_t reach(uint64_t N, uint64_t tile) { return (N + tile - 1) / tile * tile; }
inline int pick_tile(int product, int type, uint64_t M, uint64_t N, uint64_t K, int cus, bool large, bool whole)
{
    const uint64_t c = cus, t256 = tiles_of(M, N, 2);
    if (large && whole && t256 >= c &&
        (product == FWD ? N > 128 && (K >= 1024 || (K >= 256 && t256 >= 4 * c)) : reach(N, 256) * 4 <= reach(N, 128) * 5)) return 2;
    if (large && product == FWD && N > 128 && tiles_of(M, N, 4) * 4 >= 3 * c) return 4;
    return type != OPAL_F32 && K >= 512 && tiles_of(M, N, 1) * 2 >= 3 * c && reach(N, 128) * 4 <= reach(N, 64) * 5 ? 1 : 0;
}

// The kernel for few rows, while its blocks (64 x 16 results, all of k) find a CU each (rows x N x K): 16-bit types 64 x 512 x 1564 8.1 us against 10.3
// with 64 x 64 tiles, 1024 rows 12.6 against 10.7; an input gradient, which gathers W's columns there one by one, up to 16 rows (9.9
// against 10.5; 100 rows 13.5 against 10.9).  32-bit types, whose tiles are bound by a wave's chain of MFMAs, both: 512 x 512 x 1564 19
// against 36, input gradients of 2048 x 100 x 356 6.4 against 10.5; 600 x 1000 x 4000 (630 blocks) 128 against 86.
inline bool few_rows(int product, int type, uint64_t M, uint64_t N, int cus)
{
    if (product == GIN && M > 16 && type != OPAL_F32) return false;
    return ((M + 63) / 64) * ((N + 15) / 16) <= (uint64_t)cus;
}

// The tile of FWD and GIN (pick_tile's arguments)
inline int product_tile(int product, int type, uint64_t M, uint64_t N, uint64_t K, int cus, bool large, bool whole)
{
    return few_rows(product, type, M, N, cus) ? 3 : pick_tile(product, type, M, N, K, cus, large, whole);
}

// Splits of the sum over the rows, none empty.  256 x 256 tiles: as many as give the 256 CUs a tile each, of at least 16 steps.
// Smaller ones: two blocks per CU, of at least four steps; 128 x 128 from twelve on: 20 000 x 512 x 512 (16 tiles) 16.3 us against 22.3 with 64 x
// 64, 6000 x 1564 x 512 (52) 16.8 against 22.0; below it 8192 x 512 x 256 (8) 9.2 against 7.1, 20 000 x 355 x 128 (3) 12.1 against 7.5.  32-bit types from 6000
// steps of all tiles together on, and not where they reach a quarter further: 100 000 x 1564 x 512 (162 500) 1389 against 1706, 6000 x 1564 x 512 (9776)
// 98 against 109, 4096 x 1564 x 512 (6656) 75 against 77, 16 384 x 356 x 512 (6144) 65 against 64 (rows not on 16 bytes: 95 against 122); below it 6000 x
// 356 x 512 (2256) 35 against 30, 3000 x 520 x 400 (1880) 36 against 23; 50 000 x 130 x 1564, a third further, 335 against 292.  Few rows, while 32 x 32 tiles find a CU each, are one block's for all of the
// sum, without splits to add up: 1999 x 355 x 63 (rows, in, out) 6.0 us a call with operands in the caches (8.7 from memory)
// against 4.8 and 4.6 for the splits' sum; 4096 x 355 x 128 8.8 against
// 10.2 + 4.6, 8192 x 355 x 128 26 against 10.6 + 4.6; 32-bit types, whose operands are loads of one column, 1024 x 512 x 512 10.0 against 13.6 +
// 4.6, 1024 x 384 x 64 9.8 against 5.5 + 4.6, 1999 x 355 x 63 15.7 against 5.9 + 4.6.  The choice does not look at the operands' alignment, so that the workspace
// does not depend on it; unaligned operands take 128 x 128 tiles in the same splits.  256 x 256 tiles ask for chunks ahead of the first step and need one: a
// sum over no rows is the small tiles', which look first.
struct Splits { int tile; uint64_t splits, rows; };
inline Splits weight_splits(uint64_t n, uint32_t in, uint32_t out, int type)
{
    if (n <= (type == OPAL_F32 ? 1024 : 4096) && tiles_of(out, in, 5) <= 256) return {5, 1, n};
    const uint64_t step = STEP_BYTES / type_bytes(type);
    const uint64_t steps = std::max<uint64_t>((n + step - 1) / step, 1);
    const uint64_t big = tiles_of(out, in, 2);
    const bool large = n > 0 && type != OPAL_F32 && in > 128 && out > 128 && steps * big >= 16 * 128;
    const uint64_t t128 = tiles_of(out, in, 1);
    const bool middle = type == OPAL_F32 ? steps * t128 >= 6000 && t128 * 16 <= tiles_of(out, in, 0) * 5 : in > 64 && out > 64 && t128 >= 12;
    const int tile = large ? 2 : middle ? 1 : 0;
    uint64_t s = large ? std::min<uint64_t>(256 / std::min<uint64_t>(big, 256), steps / 16) : std::min<uint64_t>(512 / std::min<uint64_t>(tiles_of(out, in, tile), 512), steps / 4);
    s = std::max<uint64_t>(s, 1);
    const uint64_t per = (steps + s - 1) / s;
    return {tile, (steps + per - 1) / per, per * step};
}

}  // namespace opal_head
