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

#include "cache_batch.cuh"

namespace phx {

constexpr float TREE_LOG2E = 1.4426950408889634f;
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

// Places in front of each request, in shared memory; without a split, units
template <int THREADS> struct TreePlan {
  long long before[TREE_MAX_SPLIT_BATCH + 1];
  long long warp_sum[THREADS / 32];
  long long per_, more_;         // places of a block: per_, the first more_ one more

  // by all threads of the block; ends with a barrier
  __device__ void make(const TreeView& t) {
    const int tid = threadIdx.x, lane = tid & 31, per = (t.c.batch + THREADS - 1) / THREADS, b0 = min(tid * per, t.c.batch), b1 = min(b0 + per, t.c.batch);
    auto tiles_of = [&](int b) {
      const KeyRange k = key_range(t.c, b);
      return (long long)t.c.num_kv_heads * tree_row_tiles(t, k.rq.tokens) * (t.split ? tree_key_tiles(t, k.keys) + t.setup : 1);
    };
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
  __device__ __forceinline__ TreePiece unit(const TreeView& t, long long pos) const {
    const int b = request_at(t, pos);
    const KeyRange k = key_range(t.c, b);
    const int row_tiles = tree_row_tiles(t, k.rq.tokens), in = (int)(pos - before[b]), tiles = tree_key_tiles(t, k.keys);
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
  __device__ __forceinline__ TreePiece piece(const TreeView& t, long long pos, long long end, long long* next, long long* unit_end) const {
    const int lo = request_at(t, pos);
    const KeyRange k = key_range(t.c, lo);
    TreePiece p;
    p.b = lo;
    p.tiles = tree_key_tiles(t, k.keys);
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

phx_status tree_pool_map(CUtensorMap* map, const TreeView& t, int box_rows, std::string& err);
// tcgen05 kernel (tree_attention_sm100.cu): whether it takes the call, its tile shape, its launch
bool tree_tc_supported(const TreeView& t);
void tree_tc_shape(TreeView& t);                 // rows and keys of a tile
int tree_tc_blocks_per_sm();
phx_status tree_tc_launch(const TreeView& t, cudaStream_t stream, std::string& err);

}  // namespace phx
