// Host-side declarations shared by the translation units of the attention among the nodes of a structure.
#pragma once

#include "cgtp_device.h"
#include "cgtp_host.h"

namespace cgtp {

constexpr int kQSums = 10;     // what a piece leaves for each row besides the gradient of q (attn_impl.h, QSums)

// Buffers of the backward inside its workspace.
struct AttnScratch {
  float* delta;        // (n_q, h_q)
  f32x4* row_part;     // (n_q, h_q): a row's part of the gradient of its query's position and of its head's slope
  f32x4* key_part;     // (n_k, h_kv): of the key's position
  float* slope_part;   // (blocks, h_q)
  float* parts;        // partial results of pieces
};

// w null: forward.
void attn_launch_f32(const cgtp_attn_args& a, const AttnScratch* w, hipStream_t s);
void attn_launch_bf16(const cgtp_attn_args& a, const AttnScratch* w, hipStream_t s);
void attn_launch_f16(const cgtp_attn_args& a, const AttnScratch* w, hipStream_t s);

}  // namespace cgtp
