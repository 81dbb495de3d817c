// Which tiles, pieces and scratch memory a call of psh_grouped_linear or psh_grouped_linear_grad takes: rules on sizes, types and
// alignment alone, in plain C++, so that tests can ask which kernels a call reaches.
#pragma once

#include <cstdint>

#include "../../include/pysimhip.h"
#include "psh_parts.h"

inline bool aligned16(const void* p, int size, int64_t ld, int64_t stride = 0) {
    return ((uintptr_t)p & 15) == 0 && (ld * size) % 16 == 0 && (stride * size) % 16 == 0;
}

enum TileKind { TILE_ROWS16, TILE_64, TILE_128, TILE_128_DIRECT, TILE_256_DIRECT };

// Few rows a group (up to 24): 16 of them a tile.  64 groups of 10 rows, 1024 -> 1024, bf16: 23 to 25 us (5.4 TB/s of weights; 30 us in
// 64 x 64); 256 groups of 8 rows, 6 -> 64, fp64: 5.7 us (8.7 us), three times the shortest launch here: the search for the group, loads of single
// elements (6 inputs fill no 16-byte unit's line), one product and the store follow one another, and the waves wait for 70 % of that.
// Tiles [units][rows].  Large ones re-read the operands less often, small ones waste less where a group has few rows or a layer few
// units, and there are more of them to fill the CUs: the larger ones are for layers that have one and a half of them for every CU.
// bf16, 8 groups of about 4096 rows, 1024 -> 2048: 180 us (760 TFLOP/s) in 256 x 128 with two workgroups on a CU, of which one stores its tile
// while the other multiplies; 197 us in 256 x 256 with one on a CU; 228 us in 128 x 128; 318 us in 64 x 64 (dx 174 and 633 us).  Without its loads from memory the first takes
// 143 us, without those from LDS too 105 us.  12 groups of 2500 rows, 513 -> 257, fp32, 64 x 64: 115 us (69 TFLOP/s, the matrix pipes busy for
// two thirds of the time, a fifth of it with columns behind the 257th).
// (`in`: the rows of n_in numbers that are multiplied; `transposed`: by the weights' columns, as for the gradient of x)
inline TileKind rows_kind(const psh_linear_desc* d, bool transposed, int n_out, const void* in, int64_t ld_in) {
    const int64_t mean = d->rows / d->n_groups;
    if (mean <= 24) return TILE_ROWS16;
    if (d->dtype == PSH_BF16) {
        const int64_t across = (int64_t)d->rows / 128 + d->n_groups / 2, large = across * ((n_out + 127) / 128), huge = across * ((n_out + 255) / 256);
        if (mean >= 96 && n_out > 64 && large >= 192) {
            const bool direct = aligned16(in, 2, ld_in) && aligned16(d->weight, 2, d->ld_w, d->stride_w) && (!transposed || n_out % 8 == 0);
            return !direct ? TILE_128 : mean >= 512 && n_out > 128 && huge >= 768 ? TILE_256_DIRECT : TILE_128_DIRECT;
        }
    }
    return TILE_64;
}
inline TileKind forward_kind(const psh_linear_desc* d) { return rows_kind(d, false, d->out_dim, d->x, d->ld_x); }

// whether the weight gradient's bf16 operands can come by direct loads (dp is the caller's dy, or contiguous in the workspace)
inline bool grad_direct(const psh_linear_desc* d) {
    return (d->nonlin != PSH_NL_NONE || aligned16(d->dy, 2, d->ld_dy)) && aligned16(d->x, 2, d->ld_x) && d->out_dim % 8 == 0 && d->in_dim % 8 == 0;
}
// The weight gradient's tile: [out units][in units].  256 stands for 128 x 256, of which there are two to every 256 x 256 that is counted here and in
// grad_piece: 8 groups of about 4096 rows, 1024 -> 2048, bf16, are cut into pieces of 2048 rows and joined by 37 us of k_join, where 512 workgroups
// of whole groups would be two a CU (not measured).
inline int grad_tile(const psh_linear_desc* d, bool direct) {
    if (d->dtype != PSH_BF16 || d->out_dim <= 64 || d->in_dim <= 64) return 64;
    const int64_t tiles = (int64_t)((d->out_dim + 127) / 128) * ((d->in_dim + 127) / 128);
    const int64_t huge = (int64_t)((d->out_dim + 255) / 256) * ((d->in_dim + 255) / 256);
    if (direct && d->out_dim > 128 && d->in_dim > 128 && huge * (d->rows / 2048 + d->n_groups) >= 384) return 256;
    return tiles * (d->rows / 2048 + d->n_groups) >= 192 ? 128 : 64;
}
// rows of one piece of the weight gradient's contraction: enough pieces for about four workgroups a CU
inline int64_t grad_piece(const psh_linear_desc* d, bool direct) {
    const int t = grad_tile(d, direct);
    const int64_t tiles = (int64_t)((d->out_dim + t - 1) / t) * ((d->in_dim + t - 1) / t);
    const int64_t whole = ((int64_t)d->rows + 64) / 64 * 64;
    const int64_t wanted = t == 256 ? 512 : t == 128 ? 1024 : 2048;
    if (tiles >= wanted / 2) return whole;
    int64_t L = ((int64_t)d->rows * tiles / wanted + 63) / 64 * 64;
    if (L < 128) L = 128;
    return L < whole ? L : whole;
}

struct GradSpace { int64_t dp, part_w, part_b, total; };
// (room for the pieces of either kind of tile, so that the size can be asked for before the arrays are there)
inline GradSpace grad_space(const psh_linear_desc* d) {
    GradSpace s{};
    int64_t places = 0;
    for (int direct = 0; direct < 2; ++direct) {
        const int64_t L = grad_piece(d, direct), n = cut_places_count(d->rows, d->n_groups, L);
        if (d->rows > L && n > places) places = n;   // (else no group has a second piece)
    }
    if (d->nonlin != PSH_NL_NONE) s.dp = align256((int64_t)d->rows * d->out_dim * elem_size(d->dtype));
    if (d->dweight) s.part_w = align256(places * d->out_dim * d->in_dim * wide_size(d->dtype));
    if (d->dbias) s.part_b = align256(places * d->out_dim * wide_size(d->dtype));
    s.total = s.dp + s.part_w + s.part_b;
    return s;
}
inline TileKind grad_kind(const psh_linear_desc* d) {
    const int t = grad_tile(d, grad_direct(d));
    return t == 64 ? TILE_64 : !grad_direct(d) ? TILE_128 : t == 128 ? TILE_128_DIRECT : TILE_256_DIRECT;
}

// dp = dy f'(y) lies first in the workspace; without a nonlinearity it is dy itself
struct GradPlan {
    TileKind rows, weights;
    bool joint;          // both by one launch
};
inline GradPlan grad_plan(const psh_linear_desc* d) {
    const bool own = d->nonlin != PSH_NL_NONE;
    GradPlan p;
    p.rows = rows_kind(d, true, d->in_dim, own ? d->workspace : d->dy, own ? d->out_dim : d->ld_dy);
    p.weights = grad_kind(d);
    p.joint = d->dx && d->rows > 0 && (d->dweight || d->dbias) && p.rows == p.weights;
    return p;
}
