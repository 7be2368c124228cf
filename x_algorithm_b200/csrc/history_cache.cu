// New rows enter a paged cache: per-head RMS norm of queries and keys, rotation by position, keys and values stored in their
// pages, queries stored dense - one pass over the merged projection's output (layers.py:728-736 for its column order, layers.py:
// 52-67 for the rotation; there the norm is over all heads together, here over each).
//
//   h' = h / sqrt(mean(h^2) + eps) * gain,   (a, b) -> (a cos - b sin, b cos + a sin) over the halves a, b of h'
//
// in fp32, rounded once.  Bound by memory: each element is read once and written once, 16 bytes at a time.  key_size / 16
// threads hold one head: thread i the 8 elements from 8 i on and the 8 that the rotation pairs them with, so that norm (a
// shuffle over the head's threads) and rotation stay in registers.  A round is 32 / (key_size / 16) heads of one token, queries or keys or values; a
// warp takes four rounds that follow one another, of the queries or of keys and values, with all loads in flight before the first is used.  So gains, cosines and
// sines are the same for all heads until the token changes, and are multiplied into four factors once, x' = (x A - y B) / rms, y' = (y C + x D) / rms, and
// only the warps of keys and values look up their token's place in the cache - the request by a 32-way search in q_start, its length, the page.
// Measured: 31 k tokens' rows of 32 + 8 + 8 heads of 128 with norms 147 us = 5.4 TB/s, 16384 tokens of 8 + 8 + 8 heads of 64 25 us = 4.0 TB/s, one token 3.0 us.
#include <string>

#include "cache_batch.cuh"

namespace phx {
namespace {

constexpr int APPEND_WARPS = 4;
constexpr int APPEND_ROUNDS = 4;

// n / d for n below 2^16 or d a power of two: by a product with m = 2^32 / d rounded up
struct SmallDivisor {
  uint32_t d, m;
  SmallDivisor() = default;
  explicit SmallDivisor(uint32_t divisor) : d(divisor), m((uint32_t)((0x100000000ull + divisor - 1) / divisor)) {}
  __device__ __forceinline__ uint32_t of(uint32_t n) const { return d == 1 ? n : __umulhi(n, m); }
};
struct AppendShape {
  SmallDivisor group;               // query heads of a key head
  unsigned q_blocks, kv_blocks;     // rounds of a token's queries, keys (or values)
  unsigned q_rounds, kv_rounds;     // of all tokens
  unsigned q_warps;
};

__device__ __forceinline__ uint4 load_stream(const uint16_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ void unpack8(const uint4& v, float (&x)[8]) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { const float2 f = unpack_bf2(w[i]); x[2 * i] = f.x; x[2 * i + 1] = f.y; }
}
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack_bf2(x[0], x[1]), pack_bf2(x[2], x[3]), pack_bf2(x[4], x[5]), pack_bf2(x[6], x[7]));
}
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}

// the request that token row n belongs to: the number of offsets q_start[1 .. B] at or below n, found 32 at a time
__device__ __forceinline__ int find_request(const phx_cache_batch& c, int n, int lane) {
  int lo = 0, hi = c.batch;   // the answer is in [lo, hi]
  while (hi > lo) {
    const int step = (hi - lo + 31) / 32;
    const int at = lo + (lane + 1) * step;                     // is q_start[at] still at or below n?
    const bool below = at <= hi && c.q_start[at] <= n;
    const int cnt = __popc(__ballot_sync(0xffffffffu, below));
    lo = lo + cnt * step;
    hi = min(hi, lo + step - 1);
  }
  return min(lo, c.batch - 1);
}

template <int DH>
__global__ void __launch_bounds__(32 * APPEND_WARPS, 5) history_append_kernel(const phx_cache_batch c, const phx_append_args a, const AppendShape shape) {
  constexpr int TPH = DH / 16;                 // threads of a head
  constexpr int HPR = 32 / TPH;                // heads of a round
  const int lane = threadIdx.x & 31;
  const unsigned warp = blockIdx.x * APPEND_WARPS + (threadIdx.x >> 5);
  const bool kv = warp >= shape.q_warps;       // keys and values, or queries
  const unsigned round0 = (kv ? warp - shape.q_warps : warp) * APPEND_ROUNDS, rounds = kv ? shape.kv_rounds : shape.q_rounds;
  if (round0 >= rounds) return;
  const int group = (int)shape.group.d, e0 = (lane % TPH) * 8, heads = kv ? c.num_kv_heads : a.num_q_heads;

  // round i: token, head of this lane, whether of the values
  int token[APPEND_ROUNDS], head[APPEND_ROUNDS];
  bool value[APPEND_ROUNDS];
  uint4 lo[APPEND_ROUNDS], hi[APPEND_ROUNDS];
  {
    const unsigned per = kv ? 2 * shape.kv_blocks : shape.q_blocks;
    unsigned n = round0 / per, block = round0 - n * per;
#pragma unroll
    for (int i = 0; i < APPEND_ROUNDS; ++i) {
      value[i] = kv && block >= shape.kv_blocks;
      token[i] = (int)n;
      head[i] = (int)(value[i] ? block - shape.kv_blocks : block) * HPR + lane / TPH;
      if (round0 + i >= rounds) head[i] = heads;            // none
      const int of = kv ? head[i] : (int)shape.group.of((unsigned)head[i]), part = kv ? group + (value[i] ? 1 : 0) : head[i] - of * group;
      if (head[i] < heads) {
        const uint16_t* const src = a.qkv + (long long)n * a.qkv_stride + (of * (group + 2) + part) * DH + e0;
        lo[i] = load_stream(src); hi[i] = load_stream(src + DH / 2);
      } else {
        lo[i] = hi[i] = make_uint4(0, 0, 0, 0);
      }
      if (++block == per) { block = 0; ++n; }
    }
  }

  const bool rotary = a.cos_tab != nullptr, norm = a.q_gain != nullptr;
  float A[8], B[8], C[8], D[8];                // x' = x A - y B, y' = y C + x D
  uint16_t* out = nullptr;
  bool stored = true;
#pragma unroll
  for (int i = 0; i < APPEND_ROUNDS; ++i) {
    if (round0 + i >= rounds) break;
    const int n = token[i];
    if (i == 0 || n != token[i - 1]) {         // the same for the whole warp
      if (rotary) {
        int pos = a.positions[n];
        if (pos < 0 || pos >= a.num_positions) {
          if (lane == 0) cache_report(c, CACHE_BAD_POSITION);
          pos = max(0, min(pos, a.num_positions - 1));
        }
        load8(a.cos_tab + (long long)pos * (DH / 2) + e0, A);
        load8(a.sin_tab + (long long)pos * (DH / 2) + e0, B);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) { A[k] = 1.f; B[k] = 0.f; }
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) { C[k] = A[k]; D[k] = B[k]; }
      if (norm) {
        float gx[8], gy[8];
        const float* const gain = (kv ? a.k_gain : a.q_gain) + e0;
        load8(gain, gx); load8(gain + DH / 2, gy);
#pragma unroll
        for (int k = 0; k < 8; ++k) { A[k] *= gx[k]; D[k] *= gx[k]; B[k] *= gy[k]; C[k] *= gy[k]; }
      }
      if (kv) {
        const int b = find_request(c, n, lane);
        const CacheRequest rq = cache_request(c, b);
        const bool owned = n >= rq.row0 && n < rq.row0 + rq.tokens;
        const long long at = (long long)rq.cached + (n - rq.row0);
        const int col = owned && at < cache_columns(c) ? (int)at / c.page_size : -1, slot = (int)at - col * c.page_size;
        const int page = col >= 0 ? c.block_table[(long long)b * c.table_stride + col] : -1;
        stored = page >= 0 && page < c.num_pages;
        if (!stored && lane == 0) cache_report(c, owned ? CACHE_BAD_PAGE : CACHE_BAD_OFFSETS);
        out = c.pages + (stored ? cache_row0(c, page, 0, 0) + (long long)slot * DH : 0) + e0;
      } else {
        out = a.q_out + (long long)n * a.num_q_heads * DH + e0;
      }
    }
    if ((norm || rotary) && !value[i]) {
      float x[8], y[8];
      unpack8(lo[i], x); unpack8(hi[i], y);
      float inv = 1.0f;
      if (norm) {
        float2 ss = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < 8; k += 2) {
          ss = __ffma2_rn(make_float2(x[k], x[k + 1]), make_float2(x[k], x[k + 1]), ss);
          ss = __ffma2_rn(make_float2(y[k], y[k + 1]), make_float2(y[k], y[k + 1]), ss);
        }
        float sum = ss.x + ss.y;
#pragma unroll
        for (int o = TPH / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        inv = rsqrtf(sum * (1.0f / DH) + a.eps);
      }
#pragma unroll
      for (int k = 0; k < 8; k += 2) {
        const float2 x2 = __fmul2_rn(make_float2(x[k], x[k + 1]), make_float2(inv, inv)), y2 = __fmul2_rn(make_float2(y[k], y[k + 1]), make_float2(inv, inv));
        const float2 u = __ffma2_rn(x2, make_float2(A[k], A[k + 1]), __fmul2_rn(y2, make_float2(-B[k], -B[k + 1])));
        const float2 v = __ffma2_rn(y2, make_float2(C[k], C[k + 1]), __fmul2_rn(x2, make_float2(D[k], D[k + 1])));
        x[k] = u.x; x[k + 1] = u.y; y[k] = v.x; y[k + 1] = v.y;
      }
      lo[i] = pack8(x); hi[i] = pack8(y);
    }
    if (head[i] < heads && stored) {
      uint16_t* const to = out + (kv ? (long long)(head[i] + (value[i] ? c.num_kv_heads : 0)) * c.page_size * DH : (long long)head[i] * DH);
      *reinterpret_cast<uint4*>(to) = lo[i];
      *reinterpret_cast<uint4*>(to + DH / 2) = hi[i];
    }
  }
}

template <int DH>
cudaError_t append_launch(const phx_cache_batch& c, const phx_append_args& a, cudaStream_t stream) {
  constexpr int per_round = 32 / (DH / 16);
  AppendShape shape;
  shape.group = SmallDivisor((uint32_t)(a.num_q_heads / c.num_kv_heads));
  shape.q_blocks = (unsigned)(a.num_q_heads + per_round - 1) / per_round;
  shape.kv_blocks = (unsigned)(c.num_kv_heads + per_round - 1) / per_round;
  const long long q = (long long)c.num_tokens * shape.q_blocks, kv = 2ll * c.num_tokens * shape.kv_blocks;
  if (q + kv > 0xF0000000ll) return cudaErrorInvalidValue;
  shape.q_rounds = (unsigned)q; shape.kv_rounds = (unsigned)kv;
  shape.q_warps = (unsigned)((q + APPEND_ROUNDS - 1) / APPEND_ROUNDS);
  const unsigned warps = shape.q_warps + (unsigned)((kv + APPEND_ROUNDS - 1) / APPEND_ROUNDS);
  history_append_kernel<DH><<<(warps + APPEND_WARPS - 1) / APPEND_WARPS, 32 * APPEND_WARPS, 0, stream>>>(c, a, shape);
  return cudaGetLastError();
}

}  // namespace
}  // namespace phx

using namespace phx;

extern "C" phx_status phx_history_append_device(int32_t device, const phx_cache_batch* cache, const phx_append_args* args, void* stream) {
  auto bad = [](const char* m) { set_global_error(std::string("phx_history_append_device: ") + m); return PHX_E_ARG; };
  const char* what = cache_check(cache);
  if (*what) return bad(what);
  if (!args) return bad("null argument");
  const phx_cache_batch& c = *cache;
  const phx_append_args& a = *args;
  if (a.num_q_heads < 1 || a.num_q_heads > 4096 || a.num_q_heads % c.num_kv_heads != 0) return bad("num_q_heads must be a multiple of num_kv_heads, at most 4096");
  if ((a.cos_tab != nullptr) != (a.sin_tab != nullptr)) return bad("cos_tab and sin_tab come together");
  if ((a.q_gain != nullptr) != (a.k_gain != nullptr)) return bad("q_gain and k_gain come together");
  if (a.cos_tab && a.num_positions < 1) return bad("num_positions must be positive");
  if (a.cos_tab && (!aligned16(a.cos_tab) || !aligned16(a.sin_tab))) return bad("cos_tab and sin_tab must be 16-byte aligned");
  if (a.q_gain && (!aligned16(a.q_gain) || !aligned16(a.k_gain) || !(a.eps >= 0.f))) return bad("gains must be 16-byte aligned, eps not negative");
  const long long width = (long long)(a.num_q_heads + 2 * c.num_kv_heads) * c.key_size;
  if (a.qkv_stride < width || a.qkv_stride % 8 != 0) return bad("qkv_stride must be a multiple of 8 and cover a row");
  if (c.batch == 0 || c.num_tokens == 0) return PHX_OK;
  if (!a.qkv || !a.q_out || !aligned16(a.qkv) || !aligned16(a.q_out)) return bad("qkv and q_out must be 16-byte aligned buffers");
  if (a.cos_tab && !a.positions) return bad("positions are required with a rotation");
  DeviceScope scope(device);
  if (!scope.ok()) { set_global_error("phx_history_append_device: cudaSetDevice failed"); return PHX_E_CUDA; }
  cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = taken_back(c.key_size == 32 ? append_launch<32>(c, a, st) : c.key_size == 64 ? append_launch<64>(c, a, st) : append_launch<128>(c, a, st));
  if (e != cudaSuccess) { set_global_error(std::string("phx_history_append_device: ") + cudaGetErrorString(e)); return PHX_E_CUDA; }
  dispatch_note(DK_HISTORY_APPEND);
  return PHX_OK;
}

extern "C" phx_status phx_decode_status(int32_t device, int32_t* status_dev, void* stream, int32_t* bits_out) {
  auto fail = [](const char* m, phx_status s) { set_global_error(std::string("phx_decode_status: ") + m); return s; };
  if (!status_dev || !bits_out) return fail("null argument", PHX_E_ARG);
  *bits_out = 0;
  DeviceScope scope(device);
  if (!scope.ok()) return fail("cudaSetDevice failed", PHX_E_CUDA);
  int32_t now[4] = {0, 0, 0, 0};
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e = cudaMemcpyAsync(now, status_dev, sizeof(now), cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && (now[0] != 0 || now[2] != 0)) {
    e = cudaMemsetAsync(status_dev, 0, 4, st);
    if (e == cudaSuccess) e = cudaMemsetAsync(status_dev + 2, 0, 4, st);
  }
  if (taken_back(e) != cudaSuccess) return fail(cudaGetErrorString(e), PHX_E_CUDA);
  *bits_out = now[2];
  if (now[0] != 0) return fail("a bounded wait ran out", PHX_E_TIMEOUT);
  if (now[2] != 0) {
    std::string m = "out of range:";
    if (now[2] & CACHE_BAD_PAGE) m += " a page of the block table;";
    if (now[2] & CACHE_BAD_POSITION) m += " a position;";
    if (now[2] & CACHE_BAD_OFFSETS) m += " offsets or lengths;";
    return fail(m.c_str(), PHX_E_ARG);
  }
  return PHX_OK;
}
