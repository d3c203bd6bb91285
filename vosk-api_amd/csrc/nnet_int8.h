// The 8-bit form of a looped nnet3 plan (nnet_plan.h): which of its affine ops
// run as 8-bit products (int8_ops.h), their weights in codes, and the row
// maps that they read and write their frame rings through.
//
// An op becomes a product where its input is one affine layer's output at one
// or more time offsets (a TDNN-F layer's splice), computed at evenly spaced
// times, and its fused stages are bias, ReLU, scale + offset and one bypass,
// in that order.  The first layer keeps 32 bits: its input is assembled from
// features and an i-vector, of sizes that one scale a frame does not serve,
// and its weights are a few per cent of the model's.  A node that a product
// reads has, next to its ring of floats, a ring of codes and scales, written by
// a quantisation after the op that computes it; the rings of floats stay what
// every other op reads.
//
// Weights have one scale for each output column, activations one for each
// frame; sums are exact (int8_ops.h), so a stream's log-likelihoods do not
// depend on the batch it runs in.
#pragma once

#include <cstdint>
#include <string>
#include <vector>

#include "nnet_plan.h"

namespace vamd {

struct Int8Plan {
  // one frame_map launch: `rows` output rows a job, `step` frames apart; a
  // column is the ring row of the job's time + offset + step * i
  struct Map {
    int step = 1, rows = 1;
    std::vector<int> offsets;
  };
  struct OpPlan {
    bool product = false;
    bool quantize = false;  // the op's rows go into its node's ring of codes
    int map = -1, out_col = -1;  // (also of an op that is quantised but no product)
    int col = 0, taps = 0, node = -1, k = 0;  // product: taps columns from col on, the node's codes, padded dim
    int res_col = -1, res_node = -1, res_src = 0;
    float res_scale = 1.f;
    bool relu = false;
    int bias = -1;                     // NnetPlan::vecs
    std::vector<float> gain, shift;    // or empty
    std::vector<int8_t> w;             // [N][taps * k]
    std::vector<float> wscale;         // [N]
  };
  std::vector<OpPlan> ops;   // per NnetPlan op
  std::vector<Map> maps;
  std::vector<char> coded;   // per stored node: has a ring of codes
  int products = 0;
  int span = 0;              // frames that one job's maps span at most
  // Rows of a ring at most: a matrix whose rows a product maps (an output or a
  // bypass ring; not the log-likelihoods) is smaller than 2^31 bytes, and a
  // row's number has 31 bits.
  long long MaxRingRows(const NnetPlan& p) const;
  std::string Describe(const NnetPlan& p) const;
};

Int8Plan BuildInt8Plan(const NnetPlan& p);

// Codes and scale of one row, as quantize_rows gives them (int8_ops.h).
float QuantizeRow(const float* x, int k, int8_t* codes);

}  // namespace vamd
