// The attention weight that cached keys receive (phx_key_weights_device):
//
//   w_j <- decay w_j (a cached key; 0 for a new one) + sum over the rows i that see key j of e^(x_ij - lse_i),   x_ij = cap(q_i . k_j * scale)
//
// with lse_i the row's ln sum e^x that the attention gave: no maximum, no running sum, every key by itself.  Rows are the new tokens with the query heads of
// the key's head, as in tree_attention.cuh.
//
// The mma.sync kernel: S^T = K Q^T, 16 keys and 8 (16) rows at a time, so that a key's sum over the rows is one of registers and of the four lanes that share
// its row of the product.  A lane's 16-byte loads of K and Q are its fragments as they are: the product sums over the columns, in any order that both sides
// share.  K goes from memory to registers, two tiles of a warp on their way; nothing is shared between warps.
// Bound by memory and by a tile's round trips: pages, keys and old weights.  96 single tokens over up to 4096 keys, 4 key heads of 128 (273 MB): 56 us = 4.9 TB/s.  A warp's pages are asked for
// at once and old weights with the keys: 66 us without.  Tiles of a warp 4, 8, 16: 66, 55, 59 us; four warps a block for eight 55.0 and 55.7, but one token over 128 keys 3.7 and 3.1.
// That cut, 1024 keys a block, is for many users.  One token of a single user pays a warp's eight tiles in a row, eight and two tiles of a warp: over 1 k, 4 k, 16 k, 100 k keys 9.9, 10.2, 10.4, 27.9 and 4.3, 4.6,
// 5.5, 27.7 us (4 key heads of 128), 9.1, 9.2, 9.6, 33.7 and 4.1, 4.2, 7.9, 40.4 (8 of 64); 16 and 96 users of 4 k keys each 16.1, 80.7 and 20.5, 95.9 (23.6, 118.6 and 28.7, 155.4).
#include <math.h>

#include <string>

#include "tree_attention.cuh"
#include "key_weights.cuh"

namespace phx {
namespace {

constexpr int KW_WARPS = 8, KW_KEYS = 16, KW_PER = 8;   // tiles of a warp
constexpr int KW_BLOCK_TILES = KW_WARPS * KW_PER;

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 load_once(const uint16_t* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// NB blocks of 8 rows at a time; more rows than those are taken in turns
template <int DH, int CAP, int NB>
__global__ void __launch_bounds__(32 * KW_WARPS, DH == 128 && NB == 2 ? 1 : 2) key_weights_mma_kernel(const WeightsView t) {
  constexpr int CH = DH / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane >> 2, in = lane & 3, b = blockIdx.z, h = blockIdx.y, group = t.group;
  const KeyRange kr = key_range(t.c, b);
  const CacheRequest& rq = kr.rq;
  if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) {
    if (!rq.ok) cache_report(t.c, CACHE_BAD_OFFSETS);
    if (kr.keys < (long long)rq.cached + rq.tokens) cache_report(t.c, CACHE_BAD_PAGE);
  }
  const WeightCap cap(t);
  const int rows = rq.tokens * group;
  // tiles of 16 keys, without those between the first keys and the first token's window - unless their weights fade
  const int tiles = (kr.keys + KW_KEYS - 1) / KW_KEYS;
  int sinks = tiles, first = tiles;
  if (t.decay == 1.0f) {
    sinks = min(tiles, t.sinks > 0 ? (t.sinks - 1) / KW_KEYS + 1 : 0);
    first = max(sinks, max(0, rq.cached - t.window + 1) / KW_KEYS);
  }
  const int count = sinks + max(0, tiles - first);
  if (rows == 0 && t.decay == 1.0f) return;
  const bool many = rows > NB * 8;

  struct Rows { uint4 q[NB][CH]; float lse[NB][2]; int pre[NB][2], behind[NB][2]; } r;
  int pre_lo, pre_hi, behind_least, behind_last;
  auto load_rows = [&](int r0) {
    pre_lo = 0x7fffffff; pre_hi = -1; behind_least = 0x7fffffff; behind_last = -0x7fffffff;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      {
        const int row = min(r0 + n * 8 + quad, rows - 1), tok = row / group, head = h * group + row - tok * group;
        const uint16_t* q = t.a.q + (long long)(rq.row0 + tok) * t.a.q_stride + head * DH + in * 8;
#pragma unroll
        for (int c = 0; c < CH; ++c) r.q[n][c] = *reinterpret_cast<const uint4*>(q + c * 32);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = r0 + n * 8 + in * 2 + i, at = min(row, rows - 1), tok = at / group, head = h * group + at - tok * group;
        const float lse = t.lse[(long long)(rq.row0 + tok) * t.a.num_q_heads + head];
        r.lse[n][i] = row < rows ? lse * TREE_LOG2E : INFINITY;   // no row: the last one again, with no weight
        r.pre[n][i] = isinf(lse) ? -1 : span_of(t, rq, tok).x;    // a row that saw nothing, or that the caller leaves out
        r.behind[n][i] = place_of(t, rq, tok) - t.window;
        if (r.pre[n][i] >= 0) {
          pre_lo = min(pre_lo, r.pre[n][i]); pre_hi = max(pre_hi, r.pre[n][i]);
          behind_least = min(behind_least, r.behind[n][i]); behind_last = max(behind_last, r.behind[n][i]);
        } else {
          pre_lo = -1;                                      // a row that adds nothing: no tile is seen by all
        }
      }
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {                       // the other rows are the quad's other lanes'
      pre_lo = min(pre_lo, __shfl_xor_sync(0xffffffffu, pre_lo, o)); pre_hi = max(pre_hi, __shfl_xor_sync(0xffffffffu, pre_hi, o));
      behind_least = min(behind_least, __shfl_xor_sync(0xffffffffu, behind_least, o)); behind_last = max(behind_last, __shfl_xor_sync(0xffffffffu, behind_last, o));
    }
  };

  uint4 k[2][2][CH];
  int tile_of[2], page_in[2];
  float old[2];                                            // the weight of this lane's key, on its way with the keys
  int begin = blockIdx.x * KW_BLOCK_TILES + warp;
  auto tile_at = [&](int it) { const int i = begin + it * KW_WARPS; return i < count ? (i < sinks ? i : i - sinks + first) : -1; };   // of turn `it`
  int pages = -1;                                          // lane i: the page of turn i, all of them asked for at once
  auto ask_pages = [&]() { const int tile = lane < KW_PER ? tile_at(lane) : -1; if (tile >= 0) pages = kr.table[tile * KW_KEYS / t.c.page_size]; };
  auto fetch = [&](int it, int to) {
    tile_of[to] = tile_at(it);
    if (tile_of[to] < 0) return;
    const int key = tile_of[to] * KW_KEYS, page = __shfl_sync(0xffffffffu, pages, it);
    page_in[to] = page;
    if ((unsigned)page >= (unsigned)t.c.num_pages) return;
    const uint16_t* src = t.c.pages + cache_row0(t.c, page, 0, h) + (long long)(key % t.c.page_size + quad) * DH + in * 8;
#pragma unroll
    for (int c = 0; c < CH; ++c) { k[to][0][c] = load_once(src + c * 32); k[to][1][c] = load_once(src + 8 * DH + c * 32); }
    old[to] = in < 2 ? t.weights[((long long)page * t.c.num_kv_heads + h) * t.c.page_size + key % t.c.page_size + quad + 8 * in] : 0.f;
  };
  if (begin >= count) return;
  ask_pages();
  fetch(0, 0);
  if (!many && rows > 0) load_rows(0);
  for (;;) {
#pragma unroll
  for (int it = 0; it < KW_PER; ++it) {
    const int cur = it & 1;
    if (it + 1 < KW_PER) fetch(it + 1, cur ^ 1);
    if (tile_of[cur] < 0) break;
    const int page = page_in[cur];
    if ((unsigned)page >= (unsigned)t.c.num_pages) { if (lane == 0) cache_report(t.c, CACHE_BAD_PAGE); continue; }
    const int key0 = tile_of[cur] * KW_KEYS;
    // this lane's two keys
    int2 span[2];
    int place[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int key = key0 + quad + 8 * i;
      span[i] = make_int2(0, 0x7fffffff); place[i] = 0;
      if (key >= kr.keys) span[i] = make_int2(0x7fffffff, -1);
      else { if (key >= rq.cached) span[i] = span_of(t, rq, key - rq.cached); place[i] = key_place(t, rq, key); }
    }
    float sum[2] = {0.f, 0.f};
    for (int r0 = 0; r0 < rows; r0 += NB * 8) {
      if (many) {
        if (is_chain(t)) {                                  // rows in front of the tile's keys, or whose windows lie behind it
          const int tok0 = r0 / group, tok1 = min(r0 + NB * 8 - 1, rows - 1) / group;
          if (key0 > rq.cached + tok1) continue;
          if (key0 + KW_KEYS - 1 <= rq.cached + tok0 - t.window && key0 >= t.sinks) break;
        }
        load_rows(r0);
      }
      float s[NB][4];
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
          const uint4 lo = k[cur][0][c], hi = k[cur][1][c], q = r.q[n][c];
          mma_16816(s[n], lo.x, hi.x, lo.y, hi.y, q.x, q.y);
          mma_16816(s[n], lo.z, hi.z, lo.w, hi.w, q.z, q.w);
        }
      }
      const bool whole = pre_lo >= 0 && key0 + KW_KEYS <= min(rq.cached, kr.keys) && (key0 > behind_last || key0 + KW_KEYS <= t.sinks);
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        if (CAP == 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j) s[n][j] *= t.csc;
        } else if (CAP == 1) {
#pragma unroll
          for (int j = 0; j < 4; ++j) s[n][j] = cap.form.of<1>(s[n][j]);
        } else {
          cap.of_any(s[n][0], s[n][1]); cap.of_any(s[n][2], s[n][3]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int i = j >> 1, row = j & 1;
          const float p = tree_ex2(s[n][j] - r.lse[n][row]);
          const bool see = whole || (span[i].x <= r.pre[n][row] && r.pre[n][row] < span[i].y && place[i] > r.behind[n][row]);
          sum[i] += see ? p : 0.f;
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
      sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
    }
    const int key = key0 + quad + 8 * in;
    if (in < 2 && key < kr.keys) {
      float* const w = t.weights + ((long long)page * t.c.num_kv_heads + h) * t.c.page_size + key % t.c.page_size;
      *w = (key < rq.cached ? old[cur] * t.decay : 0.f) + (in == 0 ? sum[0] : sum[1]);
    }
  }
  begin += gridDim.x * KW_BLOCK_TILES;                     // requests longer than the caller said
  if (begin >= count) return;
  ask_pages();
  fetch(0, 0);
  }
}

template <int DH, int CAP, int NB>
phx_status launch_mma(const WeightsView& t, cudaStream_t stream, std::string& err) {
  long long tiles = (t.a.max_keys + KW_KEYS - 1) / KW_KEYS;
  if (t.decay == 1.0f) {
    const long long seen = ((long long)t.sinks + KW_KEYS - 1) / KW_KEYS + ((long long)t.window + t.a.max_tokens + 2 * KW_KEYS) / KW_KEYS;
    if (seen < tiles) tiles = seen;
  }
  const dim3 grid((unsigned)((tiles + KW_BLOCK_TILES - 1) / KW_BLOCK_TILES), t.c.num_kv_heads, t.c.batch);
  key_weights_mma_kernel<DH, CAP, NB><<<grid, 32 * KW_WARPS, 0, stream>>>(t);
  PHX_CUDA_TRY(cudaGetLastError(), err);
  dispatch_note(DK_KEY_WEIGHTS_MMA);
  return PHX_OK;
}
template <int DH, int CAP>
phx_status launch_rows(const WeightsView& t, cudaStream_t stream, std::string& err) {
  const long long rows = (long long)t.a.max_tokens * t.group;
  return rows <= 8 ? launch_mma<DH, CAP, 1>(t, stream, err) : launch_mma<DH, CAP, 2>(t, stream, err);
}
template <int DH>
phx_status launch(const WeightsView& t, cudaStream_t stream, std::string& err) {
  return t.a.cap_method == 0 ? launch_rows<DH, 0>(t, stream, err) : t.a.cap_method == 1 ? launch_rows<DH, 1>(t, stream, err) : launch_rows<DH, 2>(t, stream, err);
}

}  // namespace
}  // namespace phx

using namespace phx;

extern "C" phx_status phx_key_weights_device(int32_t device, const phx_cache_batch* cache, const phx_key_weights_args* args, void* stream) {
  auto bad = [](const char* m) { set_global_error(std::string("phx_key_weights_device: ") + m); return PHX_E_ARG; };
  if (!cache || !args) return bad("null argument");
  WeightsView t;
  t.c = *cache;
  // Without new tokens cached weights fade all the same, so such a call is asked for all that it reads, too
  const bool fades = args->decay != 1.0f;
  if (fades && t.c.num_tokens == 0) t.c.num_tokens = 1;
  const char* what = cache_check(&t.c);
  t.c.num_tokens = cache->num_tokens;
  if (*what) return bad(what);
  t.a.q = args->q; t.a.q_stride = args->q_stride; t.a.spans = args->spans; t.a.out = nullptr; t.a.workspace = args->workspace; t.a.workspace_bytes = args->workspace_bytes;
  t.a.max_keys = args->max_keys; t.a.max_tokens = args->max_tokens; t.a.num_q_heads = args->num_q_heads;
  t.a.sm_scale = args->sm_scale; t.a.cap = args->cap; t.a.cap_method = args->cap_method;
  t.positions = args->positions; t.lse = const_cast<float*>(args->lse); t.weights = args->weights; t.decay = args->decay;
  if (t.a.num_q_heads < 1 || t.a.num_q_heads > 4096 || t.a.num_q_heads % t.c.num_kv_heads != 0) return bad("num_q_heads must be a multiple of num_kv_heads, at most 4096");
  if (t.a.cap_method < 0 || t.a.cap_method > 2) return bad("cap_method must be 0, 1 or 2");
  if (!isfinite(t.a.sm_scale) || !isfinite(t.a.cap) || !isfinite(t.decay)) return bad("sm_scale, cap and decay must be finite");
  if (t.a.cap_method != 0 && !(t.a.cap > 0.f)) t.a.cap_method = 0;
  if (args->window < 0 || args->sinks < 0) return bad("window and sinks must not be negative");
  t.window = args->window > 0 ? args->window : 0x7fffffff;
  t.sinks = args->sinks;
  if (t.c.batch > 65535) return bad("at most 65535 requests");
  if (t.a.q_stride < (long long)t.a.num_q_heads * t.c.key_size || t.a.q_stride % 8 != 0) return bad("q_stride must be a multiple of 8 and cover a token's heads");
  if (t.a.max_tokens < 0 || t.a.max_keys < 0) return bad("negative size");
  if (t.c.batch == 0 || (t.c.num_tokens == 0 && (!fades || t.c.num_pages == 0))) return PHX_OK;
  if (t.a.max_tokens < 1) t.a.max_tokens = 1;
  if (t.a.max_tokens > t.c.num_tokens) t.a.max_tokens = t.c.num_tokens;
  if ((long long)t.c.num_tokens * t.a.num_q_heads > 2147483647ll) return bad("num_tokens x num_q_heads must fit 31 bits");
  if (t.c.num_tokens > 0 && (!t.a.q || !aligned16(t.a.q))) return bad("q must be a 16-byte aligned buffer");
  if ((t.c.num_tokens > 0 && !t.lse) || !t.weights) return bad("lse and weights are required");
  if (t.a.workspace_bytes < 0 || (t.a.workspace_bytes > 0 && (!t.a.workspace || !aligned16(t.a.workspace)))) return bad("workspace must be a 16-byte aligned buffer");
  if ((reinterpret_cast<uintptr_t>(t.a.spans) & 7) != 0) return bad("spans must be 8-byte aligned");
  if (t.c.num_pages == 0) return bad("an empty pool has no keys");
  const long long columns = (long long)t.c.table_cols * t.c.page_size;
  if (columns == 0 && t.c.num_tokens == 0) return PHX_OK;
  if (t.a.max_keys > columns) t.a.max_keys = columns;
  if (t.a.max_keys < 1) t.a.max_keys = 1;                      // no column at all: a block that reports it
  t.csc = t.a.sm_scale * TREE_LOG2E;
  t.group = t.a.num_q_heads / t.c.num_kv_heads;
  DeviceScope scope(device);
  if (!scope.ok()) { set_global_error("phx_key_weights_device: cudaSetDevice failed"); return PHX_E_CUDA; }
  std::string err;
  cudaStream_t st = (cudaStream_t)stream;
  const phx_status s = weights_tc_supported(t) ? weights_tc_launch(t, st, err) : t.c.key_size == 32 ? launch<32>(t, st, err) : t.c.key_size == 64 ? launch<64>(t, st, err) : launch<128>(t, st, err);
  if (s != PHX_OK) {
    (void)cudaGetLastError();
    set_global_error("phx_key_weights_device: " + err);
  }
  return s;
}
