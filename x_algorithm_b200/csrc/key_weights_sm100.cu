// The attention weight that cached keys receive, on Blackwell tensor cores (tcgen05 + TMEM + TMA), for requests of more than 16 query rows a key head; the semantics are
// key_weights.cu's.  S^T = K Q^T: 128 keys are the rows of the product and 256 query rows its columns, so that a key's sum over the queries is the sum along one thread's row of
// tensor memory, and no thread needs another's.  A block (one an SM) takes unit after unit - a request, key head and tile of 128 keys, with all tiles of rows or a
// chunk of them - K once, then the rows that see one of its keys, two tiles of 128 at a time (each role's own instructions a time, 1000 to 2700 cycles of a warp that is alone in its
// code, were what the block waited for at one: 8 x 1022 tokens that see themselves, 16 heads of 128, 76 us):
//   warp 0      producer: K (page by page) and Q tiles by TMA, and a note about each pair
//   warp 1      MMA issuer: S^T into one of two buffers of tensor memory
//   warp 2      planner, units ahead: where a unit's keys lie, what sees them, which tiles of rows
//   warps 3, 20 .. 22   every fourth tile of rows each: the rows' lse and what they see, which of the four groups of 32 rows see keys at all, and which not all
//   warps 4-19  thread = key and a group of the rows: e^(x - lse) summed up in a register; at the unit's end the groups hand their sums to the first, which writes the weight
//               (or a part, where chunks of rows are joined by key_weights_join_kernel)
// Waits are bounded; when one runs out the flag is raised, every later wait of any role fails at once, and a role whose wait failed is done.
#include <string.h>

#include <string>

#include "key_weights.cuh"
#include "sm100_ptx.cuh"

namespace phx {
namespace {

using namespace sm100;

constexpr int KT = 128, HT = 128, RT = 2 * HT;   // keys of a tile, rows of a tile, of a pair
constexpr int KW_FIRST = 4, KW_SETS = 4, KW_SUM = 4 * KW_SETS;   // warps 4 .. 19 sum, four for each group of 32 rows
constexpr int KW_ROWS = 4, KW_THREADS = 32 * (KW_FIRST + KW_SUM + KW_ROWS - 1);
constexpr int NK = 2, NS = 2;            // K tiles in shared memory, S^T buffers in tensor memory
__host__ __device__ constexpr int q_buffers(int dh) { return dh == 64 ? 3 : 2; }      // pairs of Q tiles
__host__ __device__ constexpr int row_buffers(int dh) { return dh == 64 ? 4 : 3; }    // pairs that are described
constexpr int NU = 4;                    // units that are planned or worked on

struct alignas(16) RowNote { float less[RT]; int2 sees[RT]; uint32_t flags[2]; };   // -lse in the log2 domain, -inf: no weight; (place in the walk or -1, place behind which the window begins)
struct KeyNote { int x, y, place, at; };            // span, place in the window's terms, word of the weights or -1: no key
constexpr uint32_t MASKED_AT = 4;                   // of RowNote.flags of a tile: bits 0-3 a row of the group sees a key, 4-7 some row does not see some key
constexpr uint32_t LAST = 1, FINAL = 2, STOP = 4;   // of PairNote.flags: the unit's last pair, the block's; behind it
struct PairNote { int tile, tiles; uint32_t flags; };   // its first tile, how many it has (0: a unit without rows)
struct UnitNote {
  int row0, tokens, cached, h;
  int x_least, x_most, y_least, y_most, place_least, place_most;   // over its keys: what a row has to be to see any, or all of them
  int begin, end;                        // tiles of rows that may see some
  int part;                              // the place of its sums among the parts
  uint32_t flags;                        // FINAL: the block's last
  uint32_t seen[2];                      // which of the first 64 of them do; those behind are looked at whether or not
  int k_row[KT / 16];                    // rows of the pool that its boxes begin at
};

template <int DH>
struct KwSmem {
  static constexpr int DCH = DH / 64, NQ = q_buffers(DH), NR = row_buffers(DH);
  uint8_t k[NK][DCH * KT * 128];
  uint8_t q[NQ][DCH * RT * 128];
  RowNote rows[NR];
  KeyNote keys[NU][KT];
  float sums[NU][KW_SETS - 1][KT];
  PairNote pair[NR];
  UnitNote unit[NU];
  uint64_t k_full[NK], k_empty[NK], q_full[NQ], q_empty[NQ], pair_known[NR], rows_full[NR], rows_empty[NR], s_full[NS], s_empty[NS], sums_full[NU], u_full[NU], u_empty[NU];
  uint32_t tmem;
  TreePlan<KW_THREADS> plan;
};

struct KwUnit { int b, h, key_tile, chunk, part; };

// The tiles of keys that rows may see; all of them where weights fade
__device__ __forceinline__ TileRange key_tiles(const WeightsView& t, const KeyRange& k) {
  const int all = (k.keys + KT - 1) / KT;
  if (t.decay != 1.0f || all == 0) return TileRange{all, all, all};
  return tile_range(t, k, 0, k.rq.tokens - 1);
}
__device__ __forceinline__ long long key_tiles_of(const WeightsView& t, const KeyRange& k) {
  if (k.rq.tokens == 0 && t.decay == 1.0f) return 0;
  const TileRange r = key_tiles(t, k);
  return r.sinks + max(0, r.end - r.first);
}

// What the join finds in front of the parts
struct PartsHead { long long units; int chunks, pad; };
__host__ __device__ constexpr long long parts_bytes(long long units, int chunks) { return (long long)sizeof(PartsHead) + units * KT * 4 * (chunks + 1); }

template <int DH, int CAP>
struct KwBlock {
  static constexpr int DCH = DH / 64, NQ = q_buffers(DH), NR = row_buffers(DH);
  static constexpr uint32_t BLK = DCH * KT * 128;
  const WeightsView& t;
  const CUtensorMap& map_q;
  const CUtensorMap& map_k;
  KwSmem<DH>& sm;
  int box, chunks;                       // chunks that a request's tiles of rows are taken in
  uint32_t tmem;

  __device__ __forceinline__ bool wait(const uint64_t& bar, int phase) const { return mbar_wait(smem_u32(&bar), (uint32_t)(phase & 1), t.c.status_dev); }

  // unit `pos` of the call
  __device__ __forceinline__ KwUnit unit_at(int pos) const {
    KwUnit u;
    const int unit = chunks == 1 ? pos : pos / chunks;
    u.chunk = pos - unit * chunks;
    u.part = unit * chunks + u.chunk;
    u.b = sm.plan.request_at(t, unit);
    const KeyRange k = key_range(t.c, u.b);
    const int in = unit - (int)sm.plan.before[u.b], tile = in / t.c.num_kv_heads;
    u.h = in - tile * t.c.num_kv_heads;
    u.key_tile = key_tiles(t, k).at(tile);
    return u;
  }

  // ---- planner (a whole warp) ----
  // A unit's chain - its place, the request's offsets, its pages, its keys' spans - is some 3 us of round trips, as long as four tiles: lanes look units up side by side, and a
  // unit's pages are asked for while the one in front of it is written down.  (In the producer that chain was what the block waited for: 32 x 512 candidates 94 us.)
  __device__ __forceinline__ void plan_units(int units) {
    const int lane = threadIdx.x & 31, boxes = KT / box, page_size = t.c.page_size, page_rows = 2 * t.c.num_kv_heads * page_size;
    const int no_row = (int)(t.c.num_pages * page_rows), per_tile = t.rows / t.group;   // tokens of a tile
    int before = 0;
    for (long long base = blockIdx.x; base < units; base += 32ll * gridDim.x, before += 32) {
      const long long of_lane = base + (long long)lane * gridDim.x;
      KwUnit unit{0, 0, 0, 0, 0};
      KeyRange range;
      range.keys = 0; range.rq.row0 = range.rq.tokens = range.rq.cached = 0;
      if (of_lane < units) { unit = unit_at((int)of_lane); range = key_range(t.c, unit.b); }
      auto from = [&](int v, int i) { return __shfl_sync(0xffffffffu, v, i); };
      auto ask = [&](int i) {                               // this lane's box of unit i: its page, -2 behind the keys
        const int key = from(unit.key_tile, i) * KT + lane * box, keys = from(range.keys, i), b = from(unit.b, i);
        return lane < boxes && key < keys ? t.c.block_table[(long long)b * t.c.table_stride + key / page_size] : -2;
      };
      int page_after = ask(0);
      const int count = __popc(__ballot_sync(0xffffffffu, of_lane < units));
      for (int i = 0; i < count; ++i) {
        const int n = before + i, page = page_after;
        if (i + 1 < count) page_after = ask(i + 1);
        const int b = from(unit.b, i), h = from(unit.h, i), key0 = from(unit.key_tile, i) * KT, chunk = from(unit.chunk, i), keys = from(range.keys, i);
        CacheRequest rq;
        rq.row0 = from(range.rq.row0, i); rq.tokens = from(range.rq.tokens, i); rq.cached = from(range.rq.cached, i);
        const int part = from(unit.part, i);
        const bool final = __shfl_sync(0xffffffffu, (int)(of_lane + gridDim.x >= units), i);
        const bool there = (unsigned)page < (unsigned)t.c.num_pages;
        if (page != -2 && !there) cache_report(t.c, CACHE_BAD_PAGE);
        if (lane == 0 && key0 == 0 && h == 0 && chunk == 0 && keys < (long long)rq.cached + rq.tokens) cache_report(t.c, CACHE_BAD_PAGE);
        const int slot0 = (key0 + lane * box) % page_size, row = there ? page * page_rows + h * page_size + slot0 : no_row;
        // this lane's four keys: what a row has to be to see all of them, or any.  What is asked for of new ones is asked for at once.
        KeyNote mine[KT / 32];
        int2 span[KT / 32];
        int new_place[KT / 32];
        const bool fresh = key0 + KT > rq.cached && rq.tokens > 0;
#pragma unroll
        for (int g = 0; g < KT / 32; ++g) {
          const int token = max(0, min(key0 + g * 32 + lane - rq.cached, rq.tokens - 1));
          span[g] = make_int2(token, rq.tokens); new_place[g] = t.a.spans ? rq.cached : rq.cached + token;
          if (fresh && t.a.spans) span[g] = reinterpret_cast<const int2*>(t.a.spans)[rq.row0 + token];
          if (fresh && t.positions) new_place[g] = t.positions[rq.row0 + token];
        }
        int x_most = -1, y_least = 0x7fffffff, place_least = 0x7fffffff, x_least = 0x7fffffff, y_most = -1, place_most = -1;
#pragma unroll
        for (int g = 0; g < KT / 32; ++g) {
          const int in = g * 32 + lane, key = key0 + in, owner = in / box;
          const int of = __shfl_sync(0xffffffffu, page, owner), slot = __shfl_sync(0xffffffffu, slot0, owner) + in - owner * box;
          const bool ok = (unsigned)of < (unsigned)t.c.num_pages && key < keys, cached = key < rq.cached;
          const int place = cached ? key : max(rq.cached, new_place[g]), at = (of * t.c.num_kv_heads + h) * page_size + slot;
          KeyNote m;
          m.x = !ok ? 0x7fffffff : cached ? 0 : span[g].x; m.y = !ok ? -1 : cached ? 0x7fffffff : span[g].y;
          m.place = !ok ? -1 : place < t.sinks ? 0x7fffffff : place;
          m.at = !ok ? -1 : cached ? at : -2 - at;          // a new key: no weight before
          x_least = min(x_least, m.x); y_most = max(y_most, m.y); place_most = max(place_most, m.place);
          x_most = max(x_most, m.x); y_least = min(y_least, m.y); place_least = min(place_least, m.place);
          mine[g] = m;
        }
        x_most = __reduce_max_sync(0xffffffffu, x_most); y_least = __reduce_min_sync(0xffffffffu, y_least); place_least = __reduce_min_sync(0xffffffffu, place_least);
        x_least = __reduce_min_sync(0xffffffffu, x_least); y_most = __reduce_max_sync(0xffffffffu, y_most); place_most = __reduce_max_sync(0xffffffffu, place_most);
        // its tiles of rows.  In a chain those in front of the keys, and those whose windows lie behind them, are not looked at.
        const int tiles = (rq.tokens + per_tile - 1) / per_tile, per = ((tiles + chunks - 1) / chunks + 1) & ~1;
        int begin = min(chunk * per, tiles), end = min(begin + per, tiles);
        if (is_chain(t)) {
          if (key0 > rq.cached) begin = max(begin, min(end, (key0 - rq.cached) / per_tile));
          if (key0 >= t.sinks) end = max(begin, (int)min((long long)end, ((long long)key0 + KT - 1 + t.window - rq.cached - 1 + per_tile) / per_tile));
        }
        // Which of them have a token that sees new keys alone, by the tokens' places.  (Looked up by the producer as it went, a round trip a tile, then some 800 cycles of one warp's
        // instructions: 8 x 1022 tokens that see themselves, 16 heads of 128, 78 us.)
        uint32_t seen[2] = {0xffffffffu, 0xffffffffu};
        if (t.a.spans && key0 >= rq.cached) {
          seen[0] = seen[1] = 0;
          const int first = begin * per_tile, last = min(min(end, begin + 64) * per_tile, rq.tokens);
          const float inverse = 1.0f / (float)per_tile;       // exact enough for quotients below 64: 8192 tokens at most
          for (int token = first + lane; token < last; token += 256) {
            int pre[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) pre[k] = t.a.spans[2ll * (rq.row0 + min(token + k * 32, rq.tokens - 1))];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const int at = token + k * 32 - first;
              int tile = (int)((float)at * inverse);
              tile += (tile + 1) * per_tile <= at ? 1 : tile * per_tile > at ? -1 : 0;
              if (first + at < last && pre[k] >= x_least && pre[k] < y_most) seen[tile >> 5] |= 1u << (tile & 31);
            }
          }
          seen[0] = __reduce_or_sync(0xffffffffu, seen[0]); seen[1] = __reduce_or_sync(0xffffffffu, seen[1]);
        }
        if (!wait(sm.u_empty[n % NU], n / NU - 1)) return;
        UnitNote& note = sm.unit[n % NU];
#pragma unroll
        for (int g = 0; g < KT / 32; ++g) sm.keys[n % NU][g * 32 + lane] = mine[g];
        if (lane < boxes) note.k_row[lane] = row;
        if (lane == 0) {
          note.row0 = rq.row0; note.tokens = rq.tokens; note.cached = rq.cached; note.h = h;
          note.x_least = x_least; note.x_most = x_most; note.y_least = y_least; note.y_most = y_most; note.place_least = place_least; note.place_most = place_most;
          note.begin = begin; note.end = end; note.part = part; note.seen[0] = seen[0]; note.seen[1] = seen[1];
          note.flags = final ? FINAL : 0u;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sm.u_full[n % NU]));
      }
    }
  }

  // ---- producer (a whole warp; one lane issues) ----
  __device__ __forceinline__ void produce() {
    const int lane = threadIdx.x & 31, boxes = KT / box, group = t.group, per_tile = t.rows / group, q_bytes = DCH * t.rows * 128;
    int j = 0;                                              // pairs so far
    for (int n = 0;; ++n) {
      if (!wait(sm.u_full[n % NU], n / NU)) return;
      const UnitNote& u = sm.unit[n % NU];
      const int row0 = u.row0, h = u.h, end = u.end;
      const uint64_t seen = (uint64_t)u.seen[1] << 32 | u.seen[0];
      const bool final = u.flags & FINAL;
      if (!wait(sm.k_empty[n % NK], n / NK - 1)) return;    // the first wait passes
      __syncwarp();
      if (elect_one()) {
        mbar_expect_tx(smem_u32(&sm.k_full[n % NK]), BLK);
        for (int p = 0; p < boxes; ++p)
          for (int c = 0; c < DCH; ++c) tma_load_2d(smem_u32(sm.k[n % NK]) + c * KT * 128 + p * box * 128, &map_k, smem_u32(&sm.k_full[n % NK]), c * 64, u.k_row[p]);
      }
      __syncwarp();
      const int first = u.begin;
      auto candidate = [&](int tile) {                        // the first tile from `tile` on that may see some
        const int in = tile - first;
        if (in >= 64) return tile;
        const uint64_t left = seen >> in;
        return left ? tile + __ffsll(left) - 1 : first + 64;
      };
      int tile = candidate(first);
      const bool rows = tile < end;                           // none: a pair without rows, which ends the unit all the same
      for (;;) {
        int next = rows ? candidate(tile + 1) : end, count = rows ? 1 : 0;
        if (rows && next == tile + 1 && next < end) { count = 2; next = candidate(tile + 2); }
        const bool more = next < end;
        if (!wait(sm.q_empty[j % NQ], j / NQ - 1)) return;
        if (!wait(sm.rows_empty[j % NR], j / NR - 1)) return;
        __syncwarp();
        if (elect_one()) {
          const int copies = max(count, 1);
          mbar_expect_tx(smem_u32(&sm.q_full[j % NQ]), copies * q_bytes);
          for (int i = 0; i < copies; ++i)
            for (int c = 0; c < DCH; ++c)
              tma_load_3d(smem_u32(sm.q[j % NQ]) + (c * RT + i * HT) * 128, &map_q, smem_u32(&sm.q_full[j % NQ]), c * 64, h * group, row0 + (rows ? tile + i : 0) * per_tile);
          sm.pair[j % NR] = PairNote{tile, count, more ? 0u : LAST | (final ? FINAL : 0u)};
          mbar_arrive(smem_u32(&sm.pair_known[j % NR]));
        }
        __syncwarp();
        ++j;
        if (!more) break;
        tile = next;
      }
      if (final) break;
    }
    if (!wait(sm.rows_empty[j % NR], j / NR - 1)) return;       // the row warp whose turn it is not
    if (lane == 0) { sm.pair[j % NR].flags = STOP; mbar_arrive(smem_u32(&sm.pair_known[j % NR])); }
  }

  // ---- the rows of every fourth tile (a whole warp) ----
  __device__ __forceinline__ void describe(int turn) {
    const int lane = threadIdx.x & 31, group = t.group, per_tile = t.rows / group;
    // this lane's rows, 32 apart: row r of a tile is token r / group, head r % group; behind the last one no token is
    int token_in[4], head_in[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int r = g * 32 + lane;
      token_in[g] = r < t.rows ? r / group : 1 << 30; head_in[g] = r % group;
    }
    int n = 0;
    for (int j = 0;; ++j) {
      if (!wait(sm.pair_known[j % NR], j / NR)) return;
      const PairNote note = sm.pair[j % NR];
      if (note.flags & STOP) return;
      const int which = (turn - 2 * j) & (KW_ROWS - 1);       // the pair's tile that is this warp's turn
      if (which < 2) {
        const int tile = note.tile + which;
        const bool there = which < note.tiles;
        const UnitNote& u = sm.unit[n % NU];
        CacheRequest rq;
        rq.row0 = u.row0; rq.cached = u.cached;
        const float* const lse0 = t.lse + (long long)rq.row0 * t.a.num_q_heads + u.h * group;
        float lse[4];
        int pre[4], behind[4];
        bool valid[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {                         // loads without a condition: all on their way at once
          const int token = (there ? tile : 0) * per_tile + token_in[g], at = max(0, min(token, u.tokens - 1));
          valid[g] = there && token < u.tokens;
          lse[g] = u.tokens > 0 ? lse0[(long long)at * t.a.num_q_heads + head_in[g]] : 0.f;
          pre[g] = t.a.spans && u.tokens > 0 ? t.a.spans[2ll * (rq.row0 + at)] : at;
          behind[g] = (t.positions && u.tokens > 0 ? max(rq.cached, t.positions[rq.row0 + at]) : t.a.spans ? rq.cached : rq.cached + at) - t.window;
        }
        uint32_t flags = 0;
        RowNote& rows = sm.rows[j % NR];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const bool live = valid[g] && pre[g] >= 0 && !isinf(lse[g]);    // no row, padding, one that saw nothing or that the caller leaves out
          const bool any = live && pre[g] >= u.x_least && pre[g] < u.y_most && u.place_most > behind[g];
          const bool all = live && u.x_most <= pre[g] && pre[g] < u.y_least && u.place_least > behind[g];
          if (__any_sync(0xffffffffu, any)) flags |= 1u << g;
          if (!__all_sync(0xffffffffu, all)) flags |= 1u << (MASKED_AT + g);
          rows.less[which * HT + g * 32 + lane] = live ? lse[g] * -TREE_LOG2E : -INFINITY;
          rows.sees[which * HT + g * 32 + lane] = make_int2(live ? pre[g] : -0x7fffffff - 1, behind[g]);
        }
        if (lane == 0) rows.flags[which] = flags;
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sm.rows_full[j % NR]));
      }
      n += note.flags & LAST;
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&sm.rows_empty[j % NR]));   // the note has been read, by the warps whose turn it is not, too
    }
  }

  // ---- MMA issuer (one thread) ----
  __device__ __forceinline__ void issue() {
    constexpr uint32_t idesc_pair = make_idesc(KT, RT), idesc_one = make_idesc(KT, HT);
    int n = 0;
    bool first = true;
    for (int j = 0;; ++j) {
      if (!wait(sm.pair_known[j % NR], j / NR)) return;
      const uint32_t flags = sm.pair[j % NR].flags, idesc = sm.pair[j % NR].tiles == 2 ? idesc_pair : idesc_one;
      if (first && !wait(sm.k_full[n % NK], n / NK)) return;
      if (!wait(sm.s_empty[j % NS], j / NS - 1) || !wait(sm.q_full[j % NQ], j / NQ)) return;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < DCH; ++c) {
        const uint64_t kd = make_smem_desc(smem_u32(sm.k[n % NK]) + c * KT * 128), qd = make_smem_desc(smem_u32(sm.q[j % NQ]) + c * RT * 128);
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_bf16(tmem + (j % NS) * RT, kd + (uint64_t)(k * 2), qd + (uint64_t)(k * 2), idesc, (c | k) != 0);
      }
      umma_commit(smem_u32(&sm.q_empty[j % NQ]));
      umma_commit(smem_u32(&sm.s_full[j % NS]));
      first = flags & LAST;
      if (first) { umma_commit(smem_u32(&sm.k_empty[n % NK])); ++n; }
      if (flags & FINAL) return;
    }
  }

  // ---- sums ----
  __device__ __forceinline__ void sum_up() {
    const int warp = warp_index() - KW_FIRST, lane = threadIdx.x & 31, g = warp >> 2, in = (warp & 3) * 32 + lane;   // group g of both tiles
    const uint32_t column = tmem + ((uint32_t)((warp & 3) * 32) << 16) + g * 32;
    const WeightCap cap(t);
    const float csc = CAP ? 1.0f : t.csc;
    int n = 0;
    KeyNote key{0, 0, 0, -1};
    float sum = 0.f;
    int part = 0;
    bool first = true;
    for (int j = 0;; ++j) {
      if (!wait(sm.rows_full[j % NR], j / NR) || !wait(sm.s_full[j % NS], j / NS)) return;
      tc_fence_after();
      const PairNote note = sm.pair[j % NR];
      if (first) { key = sm.keys[n % NU][in]; part = sm.unit[n % NU].part; sum = 0.f; }
      const RowNote& rows = sm.rows[j % NR];
#pragma unroll 1
      for (int i = 0; i < note.tiles; ++i) {
        const uint32_t flags = rows.flags[i];
        if (!((flags >> g) & 1)) continue;
        float s[32];
        tmem_ld32_nowait(column + (j % NS) * RT + i * HT, reinterpret_cast<uint32_t*>(s));
        tmem_ld_wait_on(s);
        if (CAP == 1) {
#pragma unroll
          for (int k = 0; k < 32; ++k) s[k] = cap.form.template of<1>(s[k]);
        } else if (CAP == 2) {
          float most = 0.f;
#pragma unroll
          for (int k = 0; k < 32; ++k) most = fmaxf(most, fabsf(s[k]));
          if (__all_sync(0xffffffffu, cap.small(most))) {
#pragma unroll
            for (int k = 0; k < 32; k += 2) cap.of_small(s[k], s[k + 1]);
          } else {
#pragma unroll
            for (int k = 0; k < 32; k += 2) cap.of_any(s[k], s[k + 1]);
          }
        }
        const float4* const less = reinterpret_cast<const float4*>(rows.less + i * HT + g * 32);
        const float2 scale = make_float2(csc, csc);
        float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        const bool masked = (flags >> (MASKED_AT + g)) & 1;
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          const float4 l = less[k / 4];
          const float2 e0 = __ffma2_rn(make_float2(s[k], s[k + 1]), scale, make_float2(l.x, l.y)), e1 = __ffma2_rn(make_float2(s[k + 2], s[k + 3]), scale, make_float2(l.z, l.w));
          s[k] = tree_ex2(e0.x); s[k + 1] = tree_ex2(e0.y); s[k + 2] = tree_ex2(e1.x); s[k + 3] = tree_ex2(e1.y);
          if (!masked) {
            acc[0] = __fadd2_rn(acc[0], make_float2(s[k], s[k + 1]));
            acc[1] = __fadd2_rn(acc[1], make_float2(s[k + 2], s[k + 3]));
          }
        }
        if (masked) {
          const int4* const sees = reinterpret_cast<const int4*>(rows.sees + i * HT + g * 32);
#pragma unroll
          for (int k = 0; k < 32; k += 2) {
            const int4 see = sees[k / 2];
            acc[0] = __fadd2_rn(acc[0], make_float2(key.x <= see.x && see.x < key.y && key.place > see.y ? s[k] : 0.f, key.x <= see.z && see.z < key.y && key.place > see.w ? s[k + 1] : 0.f));
          }
        }
        sum += (acc[0].x + acc[1].x) + (acc[0].y + acc[1].y);
      }
      tc_fence_before();
      const bool last = note.flags & LAST;
      if (last && g > 0) { sm.sums[n % NU][g - 1][in] = sum; mbar_arrive(smem_u32(&sm.sums_full[n % NU])); }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(smem_u32(&sm.s_empty[j % NS]));
        mbar_arrive(smem_u32(&sm.rows_empty[j % NR]));
        if (last) mbar_arrive(smem_u32(&sm.u_empty[n % NU]));
      }
      if (last && g == 0) {
        if (!wait(sm.sums_full[n % NU], n / NU)) return;
#pragma unroll
        for (int k = 0; k < KW_SETS - 1; ++k) sum += sm.sums[n % NU][k][in];
        if (chunks > 1) {                                    // behind the places of the weights
          t.part[((sm.plan.all(t) + part) * KT) + in] = sum;
          if (part % chunks == 0) reinterpret_cast<int*>(t.part)[(long long)(part / chunks) * KT + in] = key.at;
        } else if (key.at != -1) {
          if (key.at >= 0) { float* const w = t.weights + key.at; *w = fmaf(*w, t.decay, sum); }
          else t.weights[-2 - key.at] = sum;
        }
      }
      first = last;
      n += last;
      if (note.flags & FINAL) return;
    }
  }
};

template <int DH, int CAP>
__global__ void __launch_bounds__(KW_THREADS, 1) key_weights_tc_kernel(const __grid_constant__ WeightsView t, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, int box) {
  extern __shared__ uint8_t smem_bytes[];
  KwSmem<DH>& sm = *reinterpret_cast<KwSmem<DH>*>(smem_bytes + ((1024u - (smem_u32(smem_bytes) & 1023u)) & 1023u));
  const int warp = warp_index();
  if (threadIdx.x == 0) {
    *gave_up() = 0;
    prefetch_map(&map_q); prefetch_map(&map_k);
    for (int i = 0; i < NK; ++i) { mbar_init(smem_u32(&sm.k_full[i]), 1); mbar_init(smem_u32(&sm.k_empty[i]), 1); }
    for (int i = 0; i < q_buffers(DH); ++i) { mbar_init(smem_u32(&sm.q_full[i]), 1); mbar_init(smem_u32(&sm.q_empty[i]), 1); }
    for (int i = 0; i < NS; ++i) { mbar_init(smem_u32(&sm.s_full[i]), 1); mbar_init(smem_u32(&sm.s_empty[i]), KW_SUM); }
    for (int i = 0; i < row_buffers(DH); ++i) { mbar_init(smem_u32(&sm.pair_known[i]), 1); mbar_init(smem_u32(&sm.rows_full[i]), 2); mbar_init(smem_u32(&sm.rows_empty[i]), KW_SUM + KW_ROWS); }
    for (int i = 0; i < NU; ++i) { mbar_init(smem_u32(&sm.sums_full[i]), KT * (KW_SETS - 1)); mbar_init(smem_u32(&sm.u_full[i]), 1); mbar_init(smem_u32(&sm.u_empty[i]), KW_SUM); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(smem_u32(&sm.tmem), NS * RT);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  sm.plan.make_of(t, [&](const KeyRange& k) { return key_tiles_of(t, k) * t.c.num_kv_heads; });
  const int chunks = parts_bytes(sm.plan.all(t), t.chunks) <= t.a.workspace_bytes ? t.chunks : 1;   // more keys than the caller said: no room for parts
  const int units = (int)sm.plan.all(t) * chunks;
  if (t.chunks > 1) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (blockIdx.x == 0 && threadIdx.x == 0) *static_cast<PartsHead*>(t.a.workspace) = PartsHead{sm.plan.all(t), chunks, 0};
  }
  if (blockIdx.x == 0)
    for (int b = threadIdx.x; b < t.c.batch; b += KW_THREADS)
      if (!cache_request(t.c, b).ok) cache_report(t.c, CACHE_BAD_OFFSETS);
  KwBlock<DH, CAP> block{t, map_q, map_k, sm, box, chunks, sm.tmem};
  if (blockIdx.x < units) {
    if (warp == 0) block.produce();
    else if (warp == 1) { if (elect_one()) block.issue(); }
    else if (warp == 2) block.plan_units(units);
    else if (warp >= KW_FIRST && warp < KW_FIRST + KW_SUM) block.sum_up();
    else block.describe(warp == 3 ? 0 : warp - (KW_FIRST + KW_SUM) + 1);
  }
  settle();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(sm.tmem, NS * RT);
  }
}

// Sums of a key's chunks of rows, in their order
__global__ void __launch_bounds__(256) key_weights_join_kernel(const WeightsView t) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const PartsHead head = *static_cast<const PartsHead*>(t.a.workspace);
  if (head.chunks == 1) return;
  const int* const at_of = reinterpret_cast<const int*>(t.part);
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < head.units * KT; i += (long long)gridDim.x * 256) {
    const int at = at_of[i];
    if (at == -1) continue;
    const float* const part = t.part + (head.units + i / KT * head.chunks) * KT + i % KT;
    float sum = 0.f;
#pragma unroll 4
    for (int c = 0; c < head.chunks; ++c) sum += part[c * KT];
    if (at >= 0) t.weights[at] = fmaf(t.weights[at], t.decay, sum);
    else t.weights[-2 - at] = sum;
  }
}

template <int DH, int CAP>
phx_status launch(const WeightsView& t, const CUtensorMap& map_q, const CUtensorMap& map_k, int box, int blocks, cudaStream_t stream, std::string& err) {
  constexpr int smem = (int)sizeof(KwSmem<DH>) + 1024;
  static_assert(smem <= 227 * 1024, "a block's shared memory");
  static SmemLimit limit;
  PHX_CUDA_TRY(limit.raise(key_weights_tc_kernel<DH, CAP>, smem), err);
  key_weights_tc_kernel<DH, CAP><<<blocks, KW_THREADS, smem, stream>>>(t, map_q, map_k, box);
  PHX_CUDA_TRY(cudaGetLastError(), err);
  dispatch_note(DK_KEY_WEIGHTS_TC);
  return PHX_OK;
}

template <int DH>
phx_status launch(const WeightsView& t, const CUtensorMap& map_q, const CUtensorMap& map_k, int box, int blocks, cudaStream_t stream, std::string& err) {
  return t.a.cap_method == 0 ? launch<DH, 0>(t, map_q, map_k, box, blocks, stream, err) : t.a.cap_method == 1 ? launch<DH, 1>(t, map_q, map_k, box, blocks, stream, err)
                                                                                                               : launch<DH, 2>(t, map_q, map_k, box, blocks, stream, err);
}

}  // namespace

bool weights_tc_supported(const WeightsView& t) { return (t.c.key_size == 64 || t.c.key_size == 128) && t.group <= HT && (long long)t.a.max_tokens * t.group > 16; }

phx_status weights_tc_launch(WeightsView& t, cudaStream_t stream, std::string& err) {
  t.rows = HT / t.group * t.group; t.keys = KT;
  int box = KT;                                    // the largest power of two that a page is a multiple of, at most a tile
  while (t.c.page_size % box != 0) box /= 2;
  CUtensorMap map_q, map_k;
  phx_status s = tree_query_map(&map_q, t, err);
  if (s == PHX_OK) s = tree_pool_map(&map_k, t, box, err);
  // Tiles of rows in chunks where units alone leave blocks idle in a last round: about six rounds then, of two pairs at least
  const WeightsView whole = t;
  const int per_tile = t.rows / t.group, sms = device_sms();
  const long long most_units = ((long long)t.c.table_cols * t.c.page_size + KT - 1) / KT * t.c.num_kv_heads;   // of a request
  const int slice = (int)(most_units * TREE_MAX_SPLIT_BATCH <= (1 << 27) ? TREE_MAX_SPLIT_BATCH : most_units < (1 << 27) ? (1 << 27) / most_units : 1);
  for (int b0 = 0; s == PHX_OK && b0 < whole.c.batch; b0 += slice) {   // as many requests as a block plans, whose units a number of 32 bits counts
    t = whole;
    t.c.batch = whole.c.batch - b0 < slice ? whole.c.batch - b0 : slice;
    t.c.q_start += b0; t.c.lengths += b0; t.c.block_table += b0 * t.c.table_stride;
    long long tiles = (t.a.max_keys + KT - 1) / KT;
    if (t.decay == 1.0f) {
      const long long seen = ((long long)t.sinks + KT - 1) / KT + ((long long)t.window + t.a.max_tokens + KT - 3) / KT + 1;
      if (seen < tiles) tiles = seen;
    }
    const long long units = tiles * t.c.num_kv_heads * t.c.batch, row_tiles = (t.a.max_tokens + per_tile - 1) / per_tile;
    t.chunks = 1;
    if (units < 4 * sms) {
      const long long pairs = (row_tiles + 1) / 2, want = (6ll * sms + units - 1) / units;
      long long per = pairs / want > 2 ? pairs / want : 2;   // pairs of a chunk
      if ((pairs + per - 1) / per > 15) per = (pairs + 14) / 15;
      t.chunks = (int)((pairs + per - 1) / per);
      while (t.chunks > 1 && parts_bytes(units, t.chunks) > t.a.workspace_bytes) --t.chunks;
    }
    t.part = reinterpret_cast<float*>(static_cast<uint8_t*>(t.a.workspace) + sizeof(PartsHead));
    const int blocks = (int)(units * t.chunks < sms ? units * t.chunks : sms);
    s = t.c.key_size == 64 ? launch<64>(t, map_q, map_k, box, blocks, stream, err) : launch<128>(t, map_q, map_k, box, blocks, stream, err);
    if (s == PHX_OK && t.chunks > 1) {
      const long long joins = (units * KT + 255) / 256;
      const cudaError_t e = launch_programmatic(key_weights_join_kernel, dim3((unsigned)(joins < 4 * sms ? joins : 4 * sms)), dim3(256), 0, stream, t);
      if (e != cudaSuccess) { err = cudaGetErrorString(e); s = PHX_E_CUDA; }
    }
  }
  return s;
}

}  // namespace phx
