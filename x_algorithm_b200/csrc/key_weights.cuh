// What the kernels behind phx_key_weights_device share.
#pragma once

#include "tree_attention.cuh"

namespace phx {

struct WeightsView : WindowView {   // lse is read here
  float* weights;                   // [num_pages][num_kv_heads][page_size]
  float decay;
  int chunks;                       // of a request's tiles of rows that different blocks take (tcgen05 kernel); above 1 their sums are joined behind
};

// cap(s * scale) in the log2 domain, two at a time.  A weight is an fp32 number that follows its logit one to one, so tanh is an odd polynomial with one coefficient more than
// TreeCap's for |z| <= 1/2 (1.3e-8 off, below fp32's rounding; reweighted least squares on Chebyshev nodes), and TreeCap's exponential form, off by 1e-7 of the cap, beyond.
struct WeightCap {
  TreeCap form;
  float c[5], small_scale;
  __device__ __forceinline__ WeightCap(const TreeView& t) : form(t) {
    const float z = t.a.sm_scale / t.a.cap, z2 = z * z, bz = t.a.sm_scale * TREE_LOG2E;
    c[0] = bz * 0.999999987f; c[1] = bz * z2 * -0.333330694f; c[2] = bz * z2 * z2 * 0.133247793f; c[3] = bz * z2 * z2 * z2 * -0.052986075f;
    c[4] = bz * z2 * z2 * z2 * z2 * 0.0171350061f;
    small_scale = fabsf(c[4]) <= TreeCap::MOST ? fabsf(z) : INFINITY;
  }
  __device__ __forceinline__ void of_small(float& s0, float& s1) const {
    auto two = [](float x) { return make_float2(x, x); };
    const float2 s = make_float2(s0, s1), s2 = __fmul2_rn(s, s);
    float2 p = __ffma2_rn(two(c[4]), s2, two(c[3]));
    p = __ffma2_rn(p, s2, two(c[2])); p = __ffma2_rn(p, s2, two(c[1])); p = __ffma2_rn(p, s2, two(c[0]));
    p = __fmul2_rn(p, s);
    s0 = p.x; s1 = p.y;
  }
  __device__ __forceinline__ bool small(float s) const { return fabsf(s) * small_scale <= TreeCap::SMALL; }
  __device__ __forceinline__ void of_any(float& s0, float& s1) const {
    const bool small0 = small(s0), small1 = small(s1);
    const float e0 = form.of<2>(s0), e1 = form.of<2>(s1);
    of_small(s0, s1);
    if (!small0) s0 = e0;
    if (!small1) s1 = e1;
  }
};

// tcgen05 kernel (key_weights_sm100.cu): whether it takes the call; its launch
bool weights_tc_supported(const WeightsView& t);
phx_status weights_tc_launch(WeightsView& t, cudaStream_t stream, std::string& err);

}  // namespace phx
