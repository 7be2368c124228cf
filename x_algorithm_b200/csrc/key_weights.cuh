// What the kernels behind phx_key_weights_device share.
#pragma once

#include "tree_attention.cuh"

namespace phx {

struct WeightsView : WindowView {   // lse is read here
  float* weights;                   // [num_pages][num_kv_heads][page_size]
  float decay;
};

}  // namespace phx
