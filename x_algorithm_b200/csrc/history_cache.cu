// New rows enter a paged cache: per-head RMS norm of queries and keys, rotation by position, keys and values stored in their
// pages, queries stored dense - one pass over the merged projection's output (layers.py:728-736 for its column order, layers.py:
// 52-67 for the rotation; there the norm is over all heads together, here over each).
//
//   h' = h / sqrt(mean(h^2) + eps) * gain,   (a, b) -> (a cos - b sin, b cos + a sin) over the halves a, b of h'
//
// in fp32, rounded once.  Bound by memory: each element is read once and written once, 16 bytes at a time.  key_size / 16
// threads hold one head: thread i the 8 elements from 8 i on and the 8 that the rotation pairs them with, so that norm
// (a shuffle over the head's threads) and rotation stay in registers.  A warp takes 4 x 32 / (key_size / 16) heads of one token with all its loads
// issued before the first is used, and reads the token's cosines once for all of them; what a head's place in the cache needs - the
// request by a 32-way search in q_start, its length, the page - is looked up under those loads.
#include <string>

#include "cache_batch.cuh"

namespace phx {
namespace {

constexpr int APPEND_WARPS = 4;
constexpr int APPEND_ROUNDS = 4;   // heads of a warp that follow one another, all loads in flight

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
__global__ void __launch_bounds__(32 * APPEND_WARPS) history_append_kernel(const phx_cache_batch c, const phx_append_args a, int chunks) {
  constexpr int TPH = DH / 16;                 // threads of a head
  constexpr int HPR = 32 / TPH;                // heads of a round
  const int lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * APPEND_WARPS + (threadIdx.x >> 5);
  const int n = (int)(item / chunks), chunk = (int)(item % chunks);
  if (n >= c.num_tokens) return;
  const int group = a.num_q_heads / c.num_kv_heads, per = group + 2, heads = c.num_kv_heads * per;
  const int head0 = chunk * (APPEND_ROUNDS * HPR) + lane / TPH, e0 = (lane % TPH) * 8;

  const uint16_t* row = a.qkv + (long long)n * a.qkv_stride + e0;
  uint4 lo[APPEND_ROUNDS], hi[APPEND_ROUNDS];
#pragma unroll
  for (int i = 0; i < APPEND_ROUNDS; ++i) {
    const int head = head0 + i * HPR;
    if (head < heads) { lo[i] = load_stream(row + head * DH); hi[i] = load_stream(row + head * DH + DH / 2); }
    else lo[i] = hi[i] = make_uint4(0, 0, 0, 0);
  }
  float cs[8], sn[8];
  const bool rotary = a.cos_tab != nullptr, norm = a.q_gain != nullptr;
  if (rotary) {
    int pos = a.positions[n];
    if (pos < 0 || pos >= a.num_positions) {
      if (lane == 0) cache_report(c, CACHE_BAD_POSITION);
      pos = max(0, min(pos, a.num_positions - 1));
    }
    load8(a.cos_tab + (long long)pos * (DH / 2) + e0, cs);
    load8(a.sin_tab + (long long)pos * (DH / 2) + e0, sn);
  }
  // the token's place in the cache
  const int b = find_request(c, n, lane);
  const CacheRequest rq = cache_request(c, b);
  const bool mine = n >= rq.row0 && n < rq.row0 + rq.tokens;
  const long long at = (long long)rq.cached + (n - rq.row0);
  const int col = (int)(at / c.page_size), slot = (int)(at - (long long)col * c.page_size);
  const int page = mine && at < cache_columns(c) ? c.block_table[(long long)b * c.table_stride + col] : -1;
  const bool stored = page >= 0 && page < c.num_pages;
  if (!stored && lane == 0) cache_report(c, mine ? CACHE_BAD_PAGE : CACHE_BAD_OFFSETS);
  uint16_t* const place = c.pages + (long long)slot * DH + e0;

#pragma unroll
  for (int i = 0; i < APPEND_ROUNDS; ++i) {
    const int head = head0 + i * HPR;
    const int kv = head / per, part = head - kv * per;         // part < group: a query head, group: the key, group + 1: the value
    if (__all_sync(0xffffffffu, head >= heads)) break;
    if (part <= group && (norm || rotary)) {
      float x[8], y[8];
      unpack8(lo[i], x); unpack8(hi[i], y);
      if (norm) {
        float ss = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k) ss += x[k] * x[k] + y[k] * y[k];
        const unsigned who = ((TPH == 32 ? 0u : (1u << TPH)) - 1u) << (lane & ~(TPH - 1));   // the head's threads: neighbours may hold a value
#pragma unroll
        for (int o = TPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(who, ss, o);
        const float inv = 1.0f / sqrtf(ss * (1.0f / DH) + a.eps);
        float gx[8], gy[8];
        const float* gain = (part == group ? a.k_gain : a.q_gain) + e0;
        load8(gain, gx); load8(gain + DH / 2, gy);
#pragma unroll
        for (int k = 0; k < 8; ++k) { x[k] *= inv * gx[k]; y[k] *= inv * gy[k]; }
      }
      if (rotary) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float u = x[k] * cs[k] - y[k] * sn[k];
          y[k] = y[k] * cs[k] + x[k] * sn[k];
          x[k] = u;
        }
      }
      lo[i] = pack8(x); hi[i] = pack8(y);
    }
    if (head < heads) {
      uint16_t* out = nullptr;
      if (part < group) out = a.q_out + ((long long)n * a.num_q_heads + kv * group + part) * DH + e0;
      else if (stored) out = place + cache_row0(c, page, part - group, kv);
      if (out) {
        *reinterpret_cast<uint4*>(out) = lo[i];
        *reinterpret_cast<uint4*>(out + DH / 2) = hi[i];
      }
    }
  }
}

template <int DH>
cudaError_t append_launch(const phx_cache_batch& c, const phx_append_args& a, cudaStream_t stream) {
  constexpr int heads_per_warp = APPEND_ROUNDS * 32 / (DH / 16);
  const int heads = a.num_q_heads + 2 * c.num_kv_heads;
  const int chunks = (heads + heads_per_warp - 1) / heads_per_warp;
  const long long warps = (long long)c.num_tokens * chunks;
  history_append_kernel<DH><<<(unsigned)((warps + APPEND_WARPS - 1) / APPEND_WARPS), 32 * APPEND_WARPS, 0, stream>>>(c, a, chunks);
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
  const cudaError_t e = c.key_size == 32 ? append_launch<32>(c, a, st) : c.key_size == 64 ? append_launch<64>(c, a, st) : append_launch<128>(c, a, st);
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
  if (e != cudaSuccess) return fail(cudaGetErrorString(e), PHX_E_CUDA);
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
