// The experts' products: one tiled kernel for rows sorted by expert, and what the host hands it.
//
//   forward        out[i, j] = sum_k left[i, k] right_e[j, k]     rows i of expert e, weights row-major: both operands lie
//                                                                 along the sum
//   row gradient   out[i, j] = sum_k left[i, k] right_e[k, j]     the weights lie across the sum
//   weight gradient out_e[i, j] = sum over e's rows r of left[r, i] right[r, j]     both operands lie across the sum
#pragma once

#include "a2a_device.h"
#include "a2a_internal.h"

namespace a2a {

enum ProductType : int { kFp8 = 0, kBf16 = 1, kF16 = 2 };
enum ProductMode : int { kForward = 0, kRowGradient = 1, kWeightGradient = 2 };
enum ProductEnd : int {
    kPlain = 0,      // the sums, rounded to the output's type
    kGated = 1,      // silu of the first half of the columns times the second half, and the projections themselves
    kGatedFp8 = 2,   // the same product in e4m3 with a scale per 128 columns
    kPartial = 3     // sums over parts of the operands' length, in float, for finish_kernel to add up
};

struct ProductArgs {
    const uint8_t *left;
    uint64_t left_stride;                                  // bytes from row to row
    const uint8_t *right;
    uint64_t right_stride, right_expert;                   // bytes from row to row, from expert to expert
    uint8_t *out;
    uint64_t out_stride, out_expert;                       // bytes
    uint8_t *projections;                                  // [rows, 2n] or null
    uint64_t projections_stride;                           // bytes
    const float *left_scale;
    uint64_t left_scale_elem, left_scale_row;              // elements
    const float *right_scale;
    uint64_t right_scale_expert, right_scale_row, right_scale_elem;   // elements, between blocks of 128
    float *out_scale;
    uint64_t out_scale_elem, out_scale_row;                // elements
    const int32_t *num_tokens;                             // [experts], null: one expert that has all rows
    uint32_t experts, padding, rows;
    uint32_t m;                                            // rows of a weight's gradient
    uint32_t n;                                            // columns of the output
    uint32_t k;                                            // length of the sums (not for the weight gradient: an expert's rows)
    uint32_t out_type;                                     // a2a_scalar_type
    uint32_t parts, part_steps;                            // kPartial: parts of the sums, the stages of each; out is [parts, rows, n]
    // set by the launch: tiles along the columns (all parts'), of a part, along a weight's rows; ceil(2^32 / d) of their divisors
    uint32_t tiles_n, tiles_of_part, tiles_m;
    uint32_t group_reciprocal, expert_reciprocal, part_reciprocal, run_reciprocal;
    uint32_t run, runs;                                    // weight gradient: tiles that a die takes in a row, how many times
};

// Tiles beside each other that share rows or columns of the operands, for the caches: so many rows of tiles are gone through column by
// column.
constexpr uint32_t kGroupRows = 8;

// The end of a product whose sums come in parts: their sum, and what its kind of end makes of it.
struct FinishArgs {
    const float *partial;                                  // [parts, rows, width]
    uint32_t parts, width;
};

struct GateGradientArgs {
    const uint8_t *grad_out, *projections;                 // [rows, n], [rows, 2n]
    uint8_t *grad_projections;                             // [rows, 2n]
    uint64_t grad_out_stride, projections_stride, grad_projections_stride;   // bytes
    const int32_t *num_tokens;
    uint32_t experts, padding, rows, n;
};

// `rows_per_expert`: what an expert is expected to have; it and the sizes choose the tile.
// `workspace`: memory for sums in parts, may be null.
hipError_t launch_forward(int type, int end, const ProductArgs &args, uint32_t rows_per_expert, uint32_t compute_units,
                          float *workspace, uint64_t workspace_bytes, hipStream_t stream);
hipError_t launch_gradient(int type, int mode, const ProductArgs &args, uint32_t rows_per_expert, uint32_t compute_units,
                           hipStream_t stream);
hipError_t launch_gate_gradient(int type, const GateGradientArgs &args, uint32_t compute_units, hipStream_t stream);

}  // namespace a2a
