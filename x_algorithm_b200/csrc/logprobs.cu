// Log probabilities of given ids, entropy and best alternatives from a row of logits (phx_token_logprobs_device):
//
//   c = cap tanh(x / cap),  d = (c - max c) / temperature,  Z = sum e^d
//   log p = d - ln Z,   entropy = ln Z - sum e^d d / Z
//
// The maximum is taken off before anything else, so that neither rows of a type's lowest value nor large logits overflow or cancel.
//
// One block per row.  The first pass keeps, per thread, a running maximum with its two sums and the largest (logit, id) key.  The top_k-th largest of the threads' keys is a lower bound of the row's top_k-th
// largest key, so the second pass, which finds the row in L2, collects the few keys at or above it.  Rows whose order defeats that
// bound (more keys than the buffer holds) take the exact bound from a radix select over the keys, a byte a pass.  Keys are distinct - the logit's order-preserving image,
// then the id, lowest first - so ties need no care and the result does not depend on the order of the atomics.
#include <math.h>

#include <string>

#include "cache_batch.cuh"

namespace phx {
namespace {

constexpr int LP_THREADS = 256;
constexpr int LP_KEEP = 2048;     // keys that the second pass may collect
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// order-preserving: larger logit, larger image; the two zeros are equal, NaN is largest
__device__ __forceinline__ uint32_t image(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned long long key_of(float x, int id) { return ((unsigned long long)image(x) << 32) | (uint32_t)~id; }

template <typename T> __device__ __forceinline__ float load_logit(const T* row, int i);
template <> __device__ __forceinline__ float load_logit<float>(const float* row, int i) { return row[i]; }
template <> __device__ __forceinline__ float load_logit<bf16>(const bf16* row, int i) { return bf2f(row[i]); }

// m = max c, z = sum of e^d, s = sum of e^d d
struct Stat { float m, z, s; };
__device__ __forceinline__ Stat join(const Stat& a, const Stat& b, float temperature) {
  Stat r;
  r.m = fmaxf(a.m, b.m);
  if (a.m != a.m || b.m != b.m) r.m = NAN;
  const float base = r.m == -INFINITY ? 0.f : r.m;
  const float da = (a.m - base) / temperature, db = (b.m - base) / temperature, fa = ex2(da * LOG2E), fb = ex2(db * LOG2E);
  r.z = a.z * fa + b.z * fb;
  r.s = (fa > 0.f ? fa * (a.s + a.z * da) : 0.f) + (fb > 0.f ? fb * (b.s + b.z * db) : 0.f);   // e^d d is 0 where e^d is
  return r;
}
__device__ __forceinline__ float capped(float x, float cap) { return cap > 0.f && x != -INFINITY ? cap * tanhf(x / cap) : x; }

template <typename T>
__global__ void __launch_bounds__(LP_THREADS) logprobs_kernel(const phx_logprobs_args a) {
  __shared__ unsigned long long keep[LP_KEEP];
  __shared__ Stat part[LP_THREADS / 32];
  __shared__ unsigned long long bound;
  __shared__ int count;
  __shared__ int hist[256];
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const T* row = static_cast<const T*>(a.logits) + (long long)r * a.stride;

  Stat st = {-INFINITY, 0.f, 0.f};
  unsigned long long best = 0;
  for (int i = tid; i < a.vocab; i += LP_THREADS) {
    const float x = load_logit<T>(row, i);
    const unsigned long long key = key_of(x, i);
    best = key > best ? key : best;
    if (x != -INFINITY) { const Stat one = {capped(x, a.cap), 1.f, 0.f}; st = join(st, one, a.temperature); }
  }
  for (int o = 16; o > 0; o >>= 1) {
    Stat other;
    other.m = __shfl_xor_sync(0xffffffffu, st.m, o); other.z = __shfl_xor_sync(0xffffffffu, st.z, o); other.s = __shfl_xor_sync(0xffffffffu, st.s, o);
    st = lane & o ? join(other, st, a.temperature) : join(st, other, a.temperature);
  }
  if (lane == 0) part[warp] = st;
  keep[tid] = best;
  if (tid == 0) { bound = 0; count = 0; }
  __syncthreads();
  st = part[0];
  for (int w = 1; w < LP_THREADS / 32; ++w) st = join(st, part[w], a.temperature);
  const float logz = logf(st.z);
  auto logp = [&](float x) {
    if (x == -INFINITY) return -INFINITY;
    return (capped(x, a.cap) - st.m) / a.temperature - logz;
  };
  if (a.entropy_out && tid == 0) a.entropy_out[r] = st.z == 0.f ? 0.f : logz - st.s / st.z;
  if (a.given_out)
    for (int i = tid; i < a.num_given; i += LP_THREADS) {
      const long long id = a.given[(long long)r * a.num_given + i];
      a.given_out[(long long)r * a.num_given + i] = id < 0 || id >= a.vocab ? 0.f : logp(load_logit<T>(row, (int)id));
    }
  if (a.top_k == 0 || (!a.top_out && !a.top_ids_out)) return;

  int above = 0;
  for (int i = 0; i < LP_THREADS; ++i) above += keep[i] > best;
  if (best != 0 && above == a.top_k - 1) bound = best;
  __syncthreads();
  auto collect = [&]() {
    const unsigned long long least = bound;
    for (int i = tid; i < a.vocab; i += LP_THREADS) {
      const unsigned long long key = key_of(load_logit<T>(row, i), i);
      if (key >= least) { const int at = atomicAdd(&count, 1); if (at < LP_KEEP) keep[at] = key; }
    }
    __syncthreads();
  };
  collect();
  if (count > LP_KEEP) {
    unsigned long long prefix = 0;
    int left = a.top_k;
    for (int shift = 56; shift >= 0; shift -= 8) {
      hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < a.vocab; i += LP_THREADS) {
        const unsigned long long key = key_of(load_logit<T>(row, i), i);
        if (shift == 56 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255], 1);
      }
      __syncthreads();
      int digit = 255;
      for (; digit > 0 && hist[digit] < left; --digit) left -= hist[digit];
      prefix |= (unsigned long long)digit << shift;
      __syncthreads();
    }
    if (tid == 0) { bound = prefix; count = 0; }
    __syncthreads();
    collect();
  }
  const int n = min(count, LP_KEEP);
  for (int i = tid; i < n; i += LP_THREADS) {
    const unsigned long long key = keep[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += keep[j] > key;
    if (rank >= a.top_k) continue;
    const int id = (int)~(uint32_t)key;
    if (a.top_ids_out) a.top_ids_out[(long long)r * a.top_k + rank] = id;
    if (a.top_out) a.top_out[(long long)r * a.top_k + rank] = logp(load_logit<T>(row, id));
  }
}

}  // namespace
}  // namespace phx

using namespace phx;

extern "C" phx_status phx_token_logprobs_device(int32_t device, const phx_logprobs_args* args, void* stream) {
  auto bad = [](const char* m) { set_global_error(std::string("phx_token_logprobs_device: ") + m); return PHX_E_ARG; };
  if (!args) return bad("null argument");
  const phx_logprobs_args& a = *args;
  if (a.rows < 0 || a.vocab < 1 || a.num_given < 0) return bad("rows and num_given must not be negative, vocab positive");
  if (a.top_k < 0 || a.top_k > PHX_LOGPROBS_MAX_TOP || a.top_k > a.vocab) return bad("top_k must be at most 128 and at most vocab");
  if (!(a.temperature > 0.f) || isinf(a.temperature)) return bad("temperature must be positive");
  if (!(a.cap == a.cap) || isinf(a.cap)) return bad("cap must be finite");
  if (a.stride < a.vocab) return bad("stride must cover a row");
  if (a.is_bf16 != 0 && a.is_bf16 != 1) return bad("is_bf16 must be 0 or 1");
  if (a.rows == 0) return PHX_OK;
  if (!a.logits || (reinterpret_cast<uintptr_t>(a.logits) & (a.is_bf16 ? 1 : 3)) != 0) return bad("logits must be a buffer of whole elements");
  if (a.num_given > 0 && a.given_out && !a.given) return bad("given is required with given_out");
  DeviceScope scope(device);
  if (!scope.ok()) { set_global_error("phx_token_logprobs_device: cudaSetDevice failed"); return PHX_E_CUDA; }
  if (a.is_bf16) logprobs_kernel<bf16><<<a.rows, LP_THREADS, 0, (cudaStream_t)stream>>>(a);
  else logprobs_kernel<float><<<a.rows, LP_THREADS, 0, (cudaStream_t)stream>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) { set_global_error(std::string("phx_token_logprobs_device: ") + cudaGetErrorString(e)); return PHX_E_CUDA; }
  dispatch_note(DK_TOKEN_LOGPROBS);
  return PHX_OK;
}
