// Host-side declarations shared by the translation units of the attention among the nodes of a structure.
#pragma once

#include "elem.h"

namespace cgtp {

// A call's arguments: rows of q, k, v and the gradient of the output start at multiples of 16 bytes, what a row has beyond dim in
// its last 16 bytes is zeros, and a tile's offsets fit 31 bits (a copy has been made of those that were not so).
struct AttnLaunch : cgtp_attn_args {
  int64_t g_node, g_head;      // elements between nodes and heads of the gradient of the output
};

constexpr int kQSums = 10;     // what a piece leaves for each row besides the gradient of q (attn_impl.h, QSums)

// Buffers of the backward inside its workspace.
struct AttnScratch {
  float* delta;        // (n_q, h_q)
  f32x4* row_part;     // (n_q, h_q): a row's part of the gradient of its query's position and of its head's slope
  f32x4* key_part;     // (n_k, h_kv): of the key's position
  float* slope_part;   // (h_q, blocks)
  float* parts;        // partial results of pieces
};

// w null: forward.  Defined in attn_impl.h, instantiated once for each type and kind of score.
template <typename T, bool BIASED, bool CAPPED>
void attn_launch(const AttnLaunch& a, const AttnScratch* w, hipStream_t s);

}  // namespace cgtp
