// What the kernels of the attention over a paged cache share: the request as they meet it, the caps, and how the work is cut.
//
// A unit is one request, key head and tile of query rows; row r of a request and key head is token r / group, head r % group of the
// head's queries.  Where units are few, the device's blocks share the tiles of keys of all units evenly instead (TreePlan): the units are laid
// out one after the other, each as its tiles behind `setup` places for what beginning one costs (a round trip for the offsets and pages, one for the
// keys, the join of the warps: as long as two tiles of 128 keys, six of 64; a block with many short units was the last to finish), and every block takes an equal stretch.  A unit that crosses such a bound is left in
// parts - rows of fp32 output that are not normalised, with their reference and sum - in the workspace, at most two a block, and tree_join_kernel joins
// them, in the order of the keys.  (Its blocks find what is to be joined in notes that the others leave: with a plan of its own and one warp for all parts of a row it took
// 30-60 us.)
#pragma once

#include <type_traits>

#include "cache_batch.cuh"

namespace phx {

constexpr float TREE_LOG2E = 1.4426950408889634f, TREE_LN2 = 0.69314718055994531f;
constexpr int TREE_MAX_SPLIT_BATCH = 1024;      // requests whose tiles the blocks may share

struct TreeView {
  phx_cache_batch c;
  phx_tree_args a;
  float csc;             // scale into the log2 domain (no cap)
  int group;             // query heads of a key head
  int rows, keys;        // of a tile
  int setup;             // places in front of a unit's tiles
  int split;             // blocks that share the tiles; 0: a block takes whole units
  int turns;             // blocks that take whole units in turns (tcgen05 kernel); 0: a block for each
  float* part_o;         // [2 split][rows][key_size]
  float2* part_ml;       // [2 split][rows]: reference (log2 domain), sum
  struct TreeJoin* join; // [split]: what block x's bound in front leaves to be joined
};
// The view of a call with a window: of the keys that a row may see, those whose place is behind the row's place - window, or in front of `sinks`, and the rows' ln sum e^x.
// (A type of its own, so that calls without one pass the kernels no more than they need.)
struct WindowView : TreeView {
  const int* positions;
  float* lse;
  int window, sinks;
  int tile_tokens, rows_tokens;   // that a tile of rows may touch, that it has where it has whole ones
};
template <class View> constexpr bool has_window = std::is_same<View, WindowView>::value;
// A unit cut by the bound between blocks x - 1 and x, the first that cuts it: block x - 1 has its first tiles, blocks x .. to - 1 the others
struct TreeJoin {
  int rows;              // 0: nothing to join here
  int to;
  int token0, row0, h;   // the request's first token row; the tile's first row of query; its key head
  int pad[3];
};

__device__ __forceinline__ float tree_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// cap(s * scale) in the log2 domain: method 1 s / (1 + |s| / cap), 2 cap tanh(s / cap) as cap (1 - 2 / (e^(2 s / cap) + 1)), good to 1e-7 of the cap: for logits that
// are not small against it, or under a cap of ordinary size.  Small ones take tanh as an odd polynomial for |z| <= SMALL (least maximum error over it, 1.3e-7, found by reweighted least squares on Chebyshev nodes), in the
// raw logit with all factors in the coefficients: on the fma pipe, two at a time, where two more special-function operations a logit bound the kernel (24 trees of 32
// over 8192 keys, 32 heads of 128: 178 us against 136 without a cap, when it was first measured)
struct TreeCap {
  static constexpr float SMALL = 0.5f, MOST = 3e38f;
  float scale, a, b, small_scale, c[4];
  __device__ __forceinline__ TreeCap(const TreeView& t) {
    const float cap = t.a.cap;
    auto finite = [](float x) { return fmaxf(-MOST, fminf(x, MOST)); };   // 0 times it is 0 under the smallest caps, too
    scale = t.a.cap_method == 0 ? t.csc : t.a.cap_method == 1 ? t.a.sm_scale : finite(t.a.sm_scale * 2.0f * TREE_LOG2E / cap);
    a = t.a.cap_method == 1 ? finite(1.0f / cap) : -2.0f * cap * TREE_LOG2E;
    b = cap * TREE_LOG2E;
    const float z = t.a.sm_scale / cap, z2 = z * z, bz = t.a.sm_scale * TREE_LOG2E;   // b z
    c[0] = bz * 0.999997676f; c[1] = bz * z2 * -0.333206551f; c[2] = bz * z2 * z2 * 0.13145145f; c[3] = bz * z2 * z2 * z2 * -0.0433724655f;
    small_scale = fabsf(c[3]) <= MOST ? fabsf(z) : INFINITY;              // no logit is small where the coefficients leave fp32
  }
  __device__ __forceinline__ void of_small(float& s0, float& s1) const {
    auto two = [](float x) { return make_float2(x, x); };
    const float2 s = make_float2(s0, s1), s2 = __fmul2_rn(s, s);
    float2 p = __ffma2_rn(two(c[3]), s2, two(c[2]));
    p = __ffma2_rn(p, s2, two(c[1])); p = __ffma2_rn(p, s2, two(c[0]));
    p = __fmul2_rn(p, s);
    s0 = p.x; s1 = p.y;
  }
  // either form of tanh, each logit by its own size alone
  __device__ __forceinline__ void of_any(float& s0, float& s1) const {
    auto pick = [](float size, float small, float large) {   // both are there: no branch around the one that is not taken
      float y;
      asm("{\n .reg .pred p;\n setp.le.f32 p, %1, %2;\n selp.f32 %0, %3, %4, p;\n}" : "=f"(y) : "f"(size), "f"(SMALL), "f"(small), "f"(large));
      return y;
    };
    const float size0 = fabsf(s0) * small_scale, size1 = fabsf(s1) * small_scale, e0 = of<2>(s0), e1 = of<2>(s1);
    of_small(s0, s1);
    s0 = pick(size0, s0, e0); s1 = pick(size1, s1, e1);
  }
  template <int METHOD> __device__ __forceinline__ float of(float s) const {
    const float v = s * scale;
    if (METHOD == 3) return v;                           // no cap, scaled in front of the mask: 0 * -inf is no mask
    if (METHOD == 1) return __fdividef(v, 1.0f + fabsf(v) * a) * TREE_LOG2E;
    return b + __fdividef(a, tree_ex2(v) + 1.0f);
  }
};

// The keys of one request and key head, as the kernels meet them
struct KeyRange {
  CacheRequest rq;
  int keys;             // cached + new, as far as the table has columns
  const int* table;     // the request's row of the table
};
__device__ __forceinline__ KeyRange key_range(const phx_cache_batch& c, int b) {
  KeyRange k;
  k.rq = cache_request(c, b);
  k.keys = (int)min((long long)k.rq.cached + k.rq.tokens, cache_columns(c));
  k.table = c.block_table + (long long)b * c.table_stride;
  return k;
}
// (pre, end) of new token j of a request
__device__ __forceinline__ int2 span_of(const TreeView& t, const CacheRequest& rq, int j) {
  return t.a.spans ? reinterpret_cast<const int2*>(t.a.spans)[rq.row0 + j] : make_int2(j, rq.tokens);
}
__device__ __forceinline__ bool odd_value(uint32_t v) { return (v & 0x7F80u) == 0x7F80u; }   // infinity or NaN in the low half
__device__ __forceinline__ bool odd_pair(uint32_t v) { return odd_value(v) || (v & 0x7F800000u) == 0x7F800000u; }

// A stretch of a unit's tiles of keys
struct TreePiece {
  int b, h, row_tile;
  int begin, end, tiles;        // of `tiles` in all; none where the stretch ends in front of them
  __device__ __forceinline__ bool whole() const { return begin == 0 && end == tiles; }
  // which of its block's two parts: the one that another block began, or the one that another ends
  __device__ __forceinline__ int part() const { return begin > 0 ? 0 : 1; }
};

__device__ __forceinline__ int tree_row_tiles(const TreeView& t, int tokens) { return (int)(((long long)tokens * t.group + t.rows - 1) / t.rows); }
__device__ __forceinline__ int tree_key_tiles(const TreeView& t, int keys) { return keys > 0 ? (keys - 1) / t.keys + 1 : 1; }
__device__ __forceinline__ int rows_tokens(const TreeView& t) { return t.rows / t.group; }
__device__ __forceinline__ int rows_tokens(const WindowView& t) { return t.rows_tokens; }
// (a tile of rows has whole tokens, or a power of two of rows)
__device__ __forceinline__ int tree_row_tiles(const WindowView& t, int tokens) {
  if (t.rows == t.rows_tokens * t.group) return (int)((uint32_t)(tokens + t.rows_tokens - 1) / (uint32_t)t.rows_tokens);
  return (int)(((long long)tokens * t.group + t.rows - 1) >> (31 - __clz(t.rows)));
}
__device__ __forceinline__ int key_shift(const WindowView& t) { return 31 - __clz(t.keys); }
__device__ __forceinline__ int tree_key_tiles(const WindowView& t, int keys) { return keys > 0 ? ((keys - 1) >> key_shift(t)) + 1 : 1; }

// The place of new token j, at which its window ends and which a window has to reach for its key to be seen
__device__ __forceinline__ int place_of(const WindowView& t, const CacheRequest& rq, int j) {
  return t.positions ? max(rq.cached, t.positions[rq.row0 + j]) : t.a.spans ? rq.cached : rq.cached + j;
}
// The same for key `key`, one that every window reaches where it is one of the first
__device__ __forceinline__ int key_place(const WindowView& t, const CacheRequest& rq, int key) {
  const int place = key < rq.cached ? key : place_of(t, rq, key - rq.cached);
  return place < t.sinks ? 0x7fffffff : place;
}
// The tiles of keys that rows of some tokens may see: [0, sinks) and [first, end).  A unit's tiles are counted without the gap.
// (t.keys is a power of two, and shifts serve: a unit begins with this in every role, and a division takes the one warp beside the busy ones a quarter of a microsecond.)
struct TileRange {
  int sinks, first, end;
  __device__ __forceinline__ int at(int i) const { return i < sinks ? i : i - sinks + first; }
};
__device__ __forceinline__ bool is_chain(const WindowView& t) { return !t.positions && !t.a.spans; }
__device__ __forceinline__ TileRange tile_range(const WindowView& t, const KeyRange& k, int token0, int token1) {   // tokens token0 .. token1
  const int shift = key_shift(t);
  TileRange r;
  r.end = tree_key_tiles(t, k.keys);
  r.sinks = min(r.end, t.sinks > 0 ? ((t.sinks - 1) >> shift) + 1 : 0);
  r.first = max(r.sinks, max(0, k.rq.cached + (is_chain(t) ? token0 : 0) - t.window + 1) >> shift);
  if (is_chain(t)) r.end = max(r.sinks, min(r.end, (int)((uint32_t)(k.rq.cached + token1) >> shift) + 1));
  return r;
}
// What TileRange needs of the row tile's tokens is set by the host where t.rows and t.group are
inline void set_tile_tokens(TreeView&) {}
inline void set_tile_tokens(WindowView& t) { t.tile_tokens = (t.rows + t.group - 2) / t.group + 1; t.rows_tokens = t.rows / t.group; }
// Tiles of a unit of this request: the most that a tile of its rows may see
__device__ __forceinline__ int unit_tiles(const TreeView& t, const KeyRange& k) { return tree_key_tiles(t, k.keys); }
__device__ __forceinline__ int unit_tiles(const WindowView& t, const KeyRange& k) {
  const TileRange r = tile_range(t, k, 0, k.rq.tokens - 1);
  const int all = r.sinks + max(0, tree_key_tiles(t, k.keys) - r.first);
  if (!is_chain(t)) return max(1, all);
  const uint32_t reach = ((uint32_t)t.window + (uint32_t)(t.tile_tokens + t.keys - 3)) >> key_shift(t);   // its windows reach over window + tile_tokens - 1 keys
  return (int)max(1u, min((uint32_t)all, r.sinks + reach + 1));
}

// Places in front of each request, in shared memory; without a split, units
template <int THREADS> struct TreePlan {
  long long before[TREE_MAX_SPLIT_BATCH + 1];
  long long warp_sum[THREADS / 32];
  long long per_, more_;         // places of a block: per_, the first more_ one more

  // by all threads of the block; ends with a barrier
  template <class View> __device__ void make(const View& t) {
    make_of(t, [&](const KeyRange& k) { return (long long)t.c.num_kv_heads * tree_row_tiles(t, k.rq.tokens) * (t.split ? unit_tiles(t, k) + t.setup : 1); });
  }
  // places(request's keys): its places
  template <class View, class Places> __device__ __forceinline__ void make_of(const View& t, Places places) {
    const int tid = threadIdx.x, lane = tid & 31, per = (t.c.batch + THREADS - 1) / THREADS, b0 = min(tid * per, t.c.batch), b1 = min(b0 + per, t.c.batch);
    auto tiles_of = [&](int b) { return places(key_range(t.c, b)); };
    long long mine = 0;
    for (int b = b0; b < b1; ++b) mine += tiles_of(b);
    long long sum = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const long long x = __shfl_up_sync(0xffffffffu, sum, o); sum += lane >= o ? x : 0; }
    if (lane == 31) warp_sum[tid >> 5] = sum;
    __syncthreads();
    long long at = sum - mine;
    for (int w = 0; w < (tid >> 5); ++w) at += warp_sum[w];
    for (int b = b0; b < b1; ++b) { before[b] = at; at += per == 1 ? mine : tiles_of(b); }
    if (tid == THREADS - 1) { before[t.c.batch] = at; if (t.split) { per_ = at / t.split; more_ = at % t.split; } }   // the last thread ends behind all
    __syncthreads();
  }
  __device__ __forceinline__ long long all(const TreeView& t) const { return before[t.c.batch]; }
  __device__ __forceinline__ long long bound(int block) const { return block * per_ + min((long long)block, more_); }
  __device__ __forceinline__ int request_at(const TreeView& t, long long pos) const {
    int lo = 0, hi = t.c.batch;                          // before[lo] <= pos < before[hi]
    while (hi - lo > 1) { const int mid = (lo + hi) / 2; if (before[mid] <= pos) lo = mid; else hi = mid; }
    return lo;
  }
  // unit `pos`
  template <class View> __device__ __forceinline__ TreePiece unit(const View& t, long long pos) const {
    const int b = request_at(t, pos);
    const KeyRange k = key_range(t.c, b);
    const int row_tiles = tree_row_tiles(t, k.rq.tokens), in = (int)(pos - before[b]), tiles = unit_tiles(t, k);
    return TreePiece{b, in / row_tiles, in % row_tiles, 0, tiles, tiles};
  }
  // the first block whose stretch begins at or behind place `pos`
  __device__ __forceinline__ int block_behind(const TreeView& t, long long pos) const {
    int lo = 0, hi = t.split;
    while (lo < hi) { const int mid = (lo + hi) / 2; if (bound(mid) < pos) lo = mid + 1; else hi = mid; }
    return lo;
  }
  // what block x's first piece, from bound(x) on, leaves to be joined
  __device__ __forceinline__ void note_join(const TreeView& t, int x, const TreePiece& pc, long long unit_end) const {
    TreeJoin j;
    j.rows = 0;
    const long long first_tile = unit_end - pc.tiles;
    if (x > 0 && bound(x) > first_tile && bound(x - 1) <= first_tile) {
      const CacheRequest rq = cache_request(t.c, pc.b);
      j.row0 = pc.row_tile * t.rows;
      j.rows = (int)min((long long)t.rows, (long long)rq.tokens * t.group - j.row0);
      j.to = block_behind(t, unit_end);
      j.token0 = rq.row0; j.h = pc.h;
    }
    t.join[x] = j;
  }
  // the piece from place `pos` on, at most to `end`; `next` is behind it, `unit_end` behind its unit
  template <class View> __device__ __forceinline__ TreePiece piece(const View& t, long long pos, long long end, long long* next, long long* unit_end) const {
    const int lo = request_at(t, pos);
    const KeyRange k = key_range(t.c, lo);
    TreePiece p;
    p.b = lo;
    p.tiles = unit_tiles(t, k);
    const long long in = pos - before[lo], unit = in / (p.tiles + t.setup), unit0 = before[lo] + unit * (p.tiles + t.setup);
    const int row_tiles = tree_row_tiles(t, k.rq.tokens);
    p.h = (int)(unit / row_tiles); p.row_tile = (int)(unit - (long long)p.h * row_tiles);
    *unit_end = unit0 + p.tiles + t.setup;
    *next = min(end, *unit_end);
    p.begin = (int)max(0ll, pos - unit0 - t.setup);
    p.end = (int)max(0ll, *next - unit0 - t.setup);
    return p;
  }
};

phx_status tree_pool_map(CUtensorMap* map, const TreeView& t, int box_rows, bool wide, std::string& err);   // wide: boxes of 64 columns for heads of 32 as well, zeros behind them
phx_status tree_query_map(CUtensorMap* map, const TreeView& t, std::string& err);
// tcgen05 kernel (tree_attention_sm100.cu): whether it takes the call, its tile shape, its launch
bool tree_tc_supported(const TreeView& t);
bool tree_tc_supported(const WindowView& t);
void tree_tc_shape(TreeView& t);                 // rows and keys of a tile
int tree_tc_blocks_per_sm();
phx_status tree_tc_launch(const TreeView& t, cudaStream_t stream, std::string& err);
phx_status tree_tc_launch(const WindowView& t, cudaStream_t stream, std::string& err);

}  // namespace phx
