// The attention weight that cached keys receive, on Blackwell tensor cores (tcgen05 + TMEM + TMA), for requests of more than 16 query rows a key head; the semantics are
// key_weights.cu's.  S^T = K Q^T: 128 keys are the rows of the product and 256 query rows its columns, so that a key's sum over the queries is the sum along one thread's row of
// tensor memory, and no thread needs another's.
//
// key_weights_plan_kernel writes down, a warp for each, the units - a request, key head and tile of 128 keys, with all tiles of 128 rows that may see them or a chunk of those - and the tiles of
// rows: their lse, what they see, and its bounds for each 32 of them.  key_weights_tc_kernel, a block an SM, takes unit after unit, K once, then its rows, two tiles at a time:
//   warp 0      producer: K (page by page) and Q tiles by TMA, what is written down about them by bulk copies
//   warp 1      MMA issuer: S^T into one of two buffers of tensor memory
//   warps 4-19  thread = key and a group of 32 rows of either tile, 16 at a time with the next ones on their way from tensor memory: e^(x - lse) summed up in a register, masked where some
//               key of the warp is not seen by some of the rows; at the unit's end the groups hand their sums to the first, which writes the weight (or a part, where chunks of rows
//               are joined by key_weights_join_kernel)
// (All of that in one kernel, by a planner warp and four that described rows, was slower: such code runs at 10 cycles an instruction, by one warp beside sixteen, and the block waited for it.
// 32 x 512 candidates over up to 1022 keys, 8 heads of 64: 62 us; 8 x 1022 tokens that see themselves, 16 heads of 128: 66 us.  Now 60 and 61, the plan, of 9 us, included, of which some
// lies under the tail of what is in front; without the sums 39.)  Bound by the sums' chains: tensor memory, multiply-add, exponential, add (special-function unit 41 and 64 %, issue 44 and 48 %).
// Sets of 32 columns for 16, in twice the registers and half the warps: 68; a polynomial for an eighth to a half of the exponentials: 62 to 67; loops unrolled over the tiles: 76 and 88.
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
constexpr int KW_THREADS = 32 * (KW_FIRST + KW_SUM);
constexpr int PLAN_THREADS = 256;
constexpr int NK = 2, NS = 2, NR = 4;    // K tiles in shared memory, S^T buffers in tensor memory, pairs whose rows are described
__host__ __device__ constexpr int q_buffers(int dh) { return dh == 128 ? 2 : 3; }      // pairs of Q tiles
constexpr int NU = 4;                    // units that are worked on

// What is written down in the workspace.  Rows: -lse in the log2 domain (-inf: no weight); (place in the walk, place behind which the window begins); for each 32 of them the least and the last
// such place (the least is INT_MIN where one adds nothing), the least and the last beginning
struct alignas(16) RowNote { float less[HT]; int2 sees[HT]; int4 bound[HT / 32]; };
struct alignas(16) UnitNote {
  int row0, cached, keys, key0, h;       // of its request, its first key, its key head
  int begin, end;                        // tiles of rows that may see some of its keys
  int part;                              // the place of its sums among the parts
  int rows;                              // the RowNote of the request's and head's first tile
  uint32_t seen[2];                      // which of its first 64 tiles do; those behind are looked at whether or not
  int pad[5];
  int k_row[KT / 16];                    // rows of the pool that its boxes begin at
  int at[KT / 16];                       // words of the weights that they begin at, -1: in no page of the pool
};
static_assert(sizeof(UnitNote) == 128 && sizeof(RowNote) % 16 == 0, "a lane a word; pieces of 16 bytes");
struct alignas(16) Head { long long units, rows_at, parts_at; int chunks, pad; };   // units without chunks; bytes from the workspace's begin to the RowNotes and the parts
constexpr long long UNITS_AT = sizeof(Head);
__host__ __device__ constexpr long long parts_bytes(long long units, int chunks) { return chunks > 1 ? units * KT * 4 * (chunks + 1) : 0; }

constexpr uint32_t LAST = 1, FINAL = 2;  // of PairNote.flags: the unit's last pair, the block's
struct PairNote { int tiles; uint32_t flags; };      // how many tiles it has (0: a unit without rows)
struct KeyNote { int x, y, place, at; };             // span, place in the window's terms, word of the weights: a new key's as -2 - word, -1: no key

// Wait for the tensor-memory loads in flight; the 16 registers are operands, so that no use of them is scheduled in front of it
__device__ __forceinline__ void wait_on_16(float* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]), "+f"(r[8]), "+f"(r[9]), "+f"(r[10]),
                 "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15])
               :: "memory");
}

// The tiles of keys that rows may see; all of them where weights fade
__device__ __forceinline__ TileRange key_tiles(const WeightsView& t, const KeyRange& k) {
  const int all = (k.keys + KT - 1) / KT;
  if (t.decay != 1.0f || all == 0) return TileRange{all, all, all};
  return tile_range(t, k, 0, k.rq.tokens - 1);
}
__device__ __forceinline__ int key_tiles_of(const WeightsView& t, const KeyRange& k) {
  if (k.rq.tokens == 0 && t.decay == 1.0f) return 0;
  const TileRange r = key_tiles(t, k);
  return r.sinks + max(0, r.end - r.first);
}
__device__ __forceinline__ int row_tiles_of(const WeightsView& t, const KeyRange& k) { const int per = t.rows / t.group; return (k.rq.tokens + per - 1) / per; }

// A unit, by a warp
__device__ void plan_unit(const WeightsView& t, int box, int chunks, int pos, const TreePlan<PLAN_THREADS>& units, const TreePlan<PLAN_THREADS>& tiles_of, UnitNote* out) {
  const int lane = threadIdx.x & 31, boxes = KT / box, page_size = t.c.page_size, per_tile = t.rows / t.group, heads = t.c.num_kv_heads;
  const int unit = pos / chunks, chunk = pos - unit * chunks, b = units.request_at(t, unit);
  const KeyRange k = key_range(t.c, b);
  const CacheRequest& rq = k.rq;
  const int in = unit - (int)units.before[b], at_tile = in / heads, h = in - at_tile * heads, key0 = key_tiles(t, k).at(at_tile) * KT;
  // its boxes: lane i has box i
  const int key = key0 + lane * box, col = key / page_size, slot0 = key - col * page_size;
  int page = -2;
  // (a box that no window reaches and no first key lies in: its page may be another request's by now)
  if (lane < boxes && key < k.keys && (t.decay != 1.0f || key + box - 1 > rq.cached - t.window || key < t.sinks)) page = k.table[col];
  const bool there = (unsigned)page < (unsigned)t.c.num_pages;
  if (page != -2 && !there) cache_report(t.c, CACHE_BAD_PAGE);
  // its tiles of rows.  In a chain those in front of the keys, and those whose windows lie behind them, are not looked at.
  const int tiles = row_tiles_of(t, k), per = ((tiles + chunks - 1) / chunks + 1) & ~1;
  int begin = min(chunk * per, tiles), end = min(begin + per, tiles);
  if (is_chain(t)) {
    if (key0 > rq.cached) begin = max(begin, min(end, (key0 - rq.cached) / per_tile));
    if (key0 >= t.sinks) end = max(begin, (int)min((long long)end, ((long long)key0 + KT - 1 + t.window - rq.cached - 1 + per_tile) / per_tile));
  }
  // Which of them have a token that sees new keys alone, by the tokens' places
  uint32_t seen0 = 0xffffffffu, seen1 = 0xffffffffu;
  if (t.a.spans && key0 >= rq.cached && rq.tokens > 0) {
    int x_least = 0x7fffffff, y_most = -1;
#pragma unroll
    for (int i = 0; i < KT; i += 32) {
      const int2 s = span_of(t, rq, min(key0 + i + lane, k.keys - 1) - rq.cached);   // of the last one again behind it
      x_least = min(x_least, s.x); y_most = max(y_most, s.y);
    }
    x_least = __reduce_min_sync(0xffffffffu, x_least); y_most = __reduce_max_sync(0xffffffffu, y_most);
    seen0 = seen1 = 0;
    const int first = begin * per_tile, last = min(min(end, begin + 64) * per_tile, rq.tokens);
    const float inverse = 1.0f / (float)per_tile;            // exact enough for quotients below 64: 8192 tokens at most
    for (int token0 = first + lane; token0 < last; token0 += 256) {   // eight round trips at once
      int pre[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) pre[k] = t.a.spans[2ll * (rq.row0 + min(token0 + k * 32, rq.tokens - 1))];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int in_chunk = token0 + k * 32 - first;
        int tile = (int)((float)in_chunk * inverse);
        tile += (tile + 1) * per_tile <= in_chunk ? 1 : tile * per_tile > in_chunk ? -1 : 0;
        if (first + in_chunk < last && pre[k] >= x_least && pre[k] < y_most) { if (tile < 32) seen0 |= 1u << tile; else seen1 |= 1u << (tile - 32); }
      }
    }
    seen0 = __reduce_or_sync(0xffffffffu, seen0); seen1 = __reduce_or_sync(0xffffffffu, seen1);
  }
  if (lane == 0) {
    out->row0 = rq.row0; out->cached = rq.cached; out->keys = k.keys; out->key0 = key0; out->h = h;
    out->begin = begin; out->end = end; out->part = unit * chunks + chunk; out->rows = (int)tiles_of.before[b] + h * tiles;
    out->seen[0] = seen0; out->seen[1] = seen1;
  }
  if (lane < KT / 16) {
    out->k_row[lane] = there ? (page * 2 * heads + h) * page_size + slot0 : (int)(t.c.num_pages * 2 * heads * page_size);   // behind the pool: zeros
    out->at[lane] = there ? (page * heads + h) * page_size + slot0 : -1;
  }
}

// A tile of rows, by a warp: 32 at a time
__device__ void plan_rows(const WeightsView& t, int pos, const TreePlan<PLAN_THREADS>& tiles_of, RowNote* out) {
  const int lane = threadIdx.x & 31, per_tile = t.rows / t.group, b = tiles_of.request_at(t, pos);
  const CacheRequest rq = cache_request(t.c, b);
  const int in = pos - (int)tiles_of.before[b], tiles = (rq.tokens + per_tile - 1) / per_tile, h = in / tiles, tile = in - h * tiles;
#pragma unroll
  for (int g = 0; g < HT / 32; ++g) {
    const int r = g * 32 + lane, token = tile * per_tile + r / t.group, at = min(token, rq.tokens - 1);
    const float lse = t.lse[(long long)(rq.row0 + at) * t.a.num_q_heads + h * t.group + r % t.group];
    const int pre = span_of(t, rq, at).x, behind = place_of(t, rq, at) - t.window;
    const bool live = r < t.rows && token < rq.tokens && pre >= 0 && !isinf(lse);   // no row, padding, one that saw nothing or that the caller leaves out
    constexpr int NONE = -0x7fffffff - 1;
    out->less[r] = live ? lse * -TREE_LOG2E : -INFINITY;
    out->sees[r] = make_int2(live ? pre : NONE, behind);
    const int4 bound = make_int4(__reduce_min_sync(0xffffffffu, live ? pre : NONE), __reduce_max_sync(0xffffffffu, live ? pre : NONE),
                                 __reduce_min_sync(0xffffffffu, live ? behind : 0x7fffffff), __reduce_max_sync(0xffffffffu, live ? behind : NONE));
    if (lane == 0) out->bound[g] = bound;
  }
}

__global__ void __launch_bounds__(PLAN_THREADS) key_weights_plan_kernel(const WeightsView t, int box) {
  __shared__ TreePlan<PLAN_THREADS> units, tiles;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  units.make_of(t, [&](const KeyRange& k) { return (long long)key_tiles_of(t, k) * t.c.num_kv_heads; });
  tiles.make_of(t, [&](const KeyRange& k) { return (long long)row_tiles_of(t, k) * t.c.num_kv_heads; });
  const long long all_units = units.all(t), all_tiles = tiles.all(t);
  // more keys than the caller said: no room for parts
  auto bytes = [&](int chunks) { return UNITS_AT + all_units * chunks * (long long)sizeof(UnitNote) + all_tiles * (long long)sizeof(RowNote) + parts_bytes(all_units, chunks); };
  const int chunks = bytes(t.chunks) <= t.a.workspace_bytes ? t.chunks : 1;
  uint8_t* const space = static_cast<uint8_t*>(t.a.workspace);
  if (bytes(chunks) > t.a.workspace_bytes) {                 // only offsets that name rows twice get here
    if (blockIdx.x == 0 && threadIdx.x == 0) { *reinterpret_cast<Head*>(space) = Head{0, 0, 0, 1, 0}; cache_report(t.c, CACHE_BAD_OFFSETS); }
    return;
  }
  const long long rows_at = UNITS_AT + all_units * chunks * (long long)sizeof(UnitNote), notes = all_units * chunks + all_tiles;
  if (blockIdx.x == 0) {
    if (threadIdx.x == 0) *reinterpret_cast<Head*>(space) = Head{all_units, rows_at, rows_at + all_tiles * (long long)sizeof(RowNote), chunks, 0};
    for (int b = threadIdx.x; b < t.c.batch; b += PLAN_THREADS) {
      const KeyRange k = key_range(t.c, b);
      if (!k.rq.ok) cache_report(t.c, CACHE_BAD_OFFSETS);
      if (k.keys < (long long)k.rq.cached + k.rq.tokens) cache_report(t.c, CACHE_BAD_PAGE);   // of a request, not of a unit: no unit need hold its first key
    }
  }
  for (long long i = blockIdx.x * (PLAN_THREADS / 32) + (threadIdx.x >> 5); i < notes; i += (long long)gridDim.x * (PLAN_THREADS / 32)) {
    if (i < all_tiles) plan_rows(t, (int)i, tiles, reinterpret_cast<RowNote*>(space + rows_at) + i);
    else plan_unit(t, box, chunks, (int)(i - all_tiles), units, tiles, reinterpret_cast<UnitNote*>(space + UNITS_AT) + (i - all_tiles));
  }
}

template <int DH>
struct KwSmem {
  static constexpr int DCH = (DH + 63) / 64, NQ = q_buffers(DH);
  uint8_t k[NK][DCH * KT * 128];
  uint8_t q[NQ][DCH * RT * 128];
  RowNote rows[NR][2];
  UnitNote unit[NU];
  float sums[NU][KW_SETS - 1][KT];
  PairNote pair[NR];
  uint64_t k_full[NK], k_empty[NK], q_full[NQ], q_empty[NQ], r_full[NR], r_empty[NR], s_full[NS], s_empty[NS], sums_full[NU], u_empty[NU];
  uint32_t tmem;
};

template <int DH, int CAP>
struct KwBlock {
  static constexpr int DCH = (DH + 63) / 64, NQ = q_buffers(DH);
  static constexpr uint32_t BLK = DCH * KT * 128;
  const WeightsView& t;
  const CUtensorMap& map_q;
  const CUtensorMap& map_k;
  KwSmem<DH>& sm;
  int box, units, chunks;
  const uint8_t* space;
  long long rows_at;
  float* parts;
  uint32_t tmem;

  __device__ __forceinline__ bool wait(const uint64_t& bar, int phase) const { return mbar_wait(smem_u32(&bar), (uint32_t)(phase & 1), t.c.status_dev); }

  // ---- producer (a whole warp; one lane issues) ----
  __device__ __forceinline__ void produce() {
    const int lane = threadIdx.x & 31, boxes = KT / box, group = t.group, per_tile = t.rows / group, q_bytes = DCH * t.rows * 128;
    const RowNote* const notes = reinterpret_cast<const RowNote*>(space + rows_at);
    const uint32_t* const words = reinterpret_cast<const uint32_t*>(space + UNITS_AT) + lane;   // a lane a word of a unit's note, the next one's on its way
    uint32_t word = words[(long long)blockIdx.x * 32];
    int j = 0, n = 0;                                       // pairs and units so far
    for (int pos = blockIdx.x; pos < units; pos += gridDim.x, ++n) {
      if (!wait(sm.u_empty[n % NU], n / NU - 1)) return;    // the first wait passes
      reinterpret_cast<uint32_t*>(&sm.unit[n % NU])[lane] = word;
      const bool final = pos + (int)gridDim.x >= units;
      if (!final) word = words[(long long)(pos + gridDim.x) * 32];
      __syncwarp();
      const UnitNote& u = sm.unit[n % NU];
      const int row0 = u.row0, h = u.h, first = u.begin, end = u.end, rows = u.rows;
      const uint64_t seen = (uint64_t)u.seen[1] << 32 | u.seen[0];
      if (!wait(sm.k_empty[n % NK], n / NK - 1)) return;
      __syncwarp();
      if (elect_one()) {
        mbar_expect_tx(smem_u32(&sm.k_full[n % NK]), BLK);
        for (int p = 0; p < boxes; ++p)
          for (int c = 0; c < DCH; ++c) tma_load_2d(smem_u32(sm.k[n % NK]) + c * KT * 128 + p * box * 128, &map_k, smem_u32(&sm.k_full[n % NK]), c * 64, u.k_row[p]);
      }
      __syncwarp();
      auto candidate = [&](int tile) {                        // the first tile from `tile` on that may see some
        const int in = tile - first;
        if (in >= 64) return tile;
        const uint64_t left = seen >> in;
        return left ? tile + __ffsll(left) - 1 : first + 64;
      };
      int tile = candidate(first);
      const bool some = tile < end;                           // none: a pair without rows, which ends the unit all the same
      for (;;) {
        int next = some ? candidate(tile + 1) : end, count = some ? 1 : 0;
        if (some && next == tile + 1 && next < end) { count = 2; next = candidate(tile + 2); }
        const bool more = next < end;
        if (!wait(sm.q_empty[j % NQ], j / NQ - 1)) return;
        if (!wait(sm.r_empty[j % NR], j / NR - 1)) return;
        __syncwarp();
        if (elect_one()) {
          sm.pair[j % NR] = PairNote{count, more ? 0u : LAST | (final ? FINAL : 0u)};   // in front of the arrivals, which publish it
          const uint32_t q_bar = smem_u32(&sm.q_full[j % NQ]), r_bar = smem_u32(&sm.r_full[j % NR]);
          const int copies = max(count, 1);
          mbar_expect_tx(q_bar, copies * q_bytes);
          for (int i = 0; i < copies; ++i)
            for (int c = 0; c < DCH; ++c) tma_load_3d(smem_u32(sm.q[j % NQ]) + (c * RT + i * HT) * 128, &map_q, q_bar, c * 64, h * group, row0 + (some ? tile + i : 0) * per_tile);
          mbar_expect_tx(r_bar, count * (int)sizeof(RowNote));
          for (int i = 0; i < count; ++i)
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                         ::"r"(smem_u32(&sm.rows[j % NR][i])), "l"(notes + rows + tile + i), "r"((uint32_t)sizeof(RowNote)), "r"(r_bar) : "memory");
        }
        __syncwarp();
        ++j;
        if (!more) break;
        tile = next;
      }
    }
  }

  // ---- MMA issuer (one thread) ----
  __device__ __forceinline__ void issue() {
    constexpr uint32_t idesc_pair = make_idesc(KT, RT), idesc_one = make_idesc(KT, HT);
    int n = 0;
    bool first = true;
    for (int j = 0;; ++j) {
      if (!wait(sm.q_full[j % NQ], j / NQ)) return;
      const PairNote note = sm.pair[j % NR];
      const uint32_t idesc = note.tiles == 2 ? idesc_pair : idesc_one;
      if (first && !wait(sm.k_full[n % NK], n / NK)) return;
      if (!wait(sm.s_empty[j % NS], j / NS - 1)) return;
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < DCH; ++c) {
        const uint64_t kd = make_smem_desc(smem_u32(sm.k[n % NK]) + c * KT * 128), qd = make_smem_desc(smem_u32(sm.q[j % NQ]) + c * RT * 128);
#pragma unroll
        for (int k = 0; k < (DH < 64 ? DH / 16 : 4); ++k) umma_bf16(tmem + (j % NS) * RT, kd + (uint64_t)(k * 2), qd + (uint64_t)(k * 2), idesc, (c | k) != 0);
      }
      umma_commit(smem_u32(&sm.q_empty[j % NQ]));
      umma_commit(smem_u32(&sm.s_full[j % NS]));
      first = note.flags & LAST;
      if (first) { umma_commit(smem_u32(&sm.k_empty[n % NK])); ++n; }
      if (note.flags & FINAL) return;
    }
  }

  // ---- sums ----
  // key `in` of a unit
  __device__ __forceinline__ KeyNote key_of(const UnitNote& u, int in) const {
    const int key = u.key0 + in, at0 = u.at[in / box], at = at0 + in % box;
    KeyNote m{0x7fffffff, -1, -1, -1};
    if (at0 < 0 || key >= u.keys) return m;
    m.x = 0; m.y = 0x7fffffff; m.place = key; m.at = at;
    if (key >= u.cached) {
      const int token = key - u.cached;
      m.at = -2 - at;
      if (t.a.spans) { const int2 s = reinterpret_cast<const int2*>(t.a.spans)[u.row0 + token]; m.x = s.x; m.y = s.y; }
      else m.x = token;
      m.place = t.positions ? max(u.cached, t.positions[u.row0 + token]) : t.a.spans ? u.cached : key;
    }
    if (m.place < t.sinks) m.place = 0x7fffffff;
    return m;
  }
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
      if (!wait(sm.r_full[j % NR], j / NR)) return;
      const PairNote note = sm.pair[j % NR];
      if (first) { key = key_of(sm.unit[n % NU], in); part = sm.unit[n % NU].part; sum = 0.f; }
      if (!wait(sm.s_full[j % NS], j / NS)) return;
      tc_fence_after();
      auto load = [&](float* s, int q) { tmem_ld16_nowait(column + (j % NS) * RT + (q >> 1) * HT + (q & 1) * 16, reinterpret_cast<uint32_t*>(s)); };   // half q & 1 of the group, tile q >> 1
      auto add = [&](float* s, int q, bool masked) {
        const RowNote& rows = sm.rows[j % NR][q >> 1];
        if (CAP == 1) {
#pragma unroll
          for (int k = 0; k < 16; ++k) s[k] = cap.form.template of<1>(s[k]);
        } else if (CAP == 2) {
          float most = 0.f;
#pragma unroll
          for (int k = 0; k < 16; ++k) most = fmaxf(most, fabsf(s[k]));
          if (__all_sync(0xffffffffu, cap.small(most))) {
#pragma unroll
            for (int k = 0; k < 16; k += 2) cap.of_small(s[k], s[k + 1]);
          } else {
#pragma unroll
            for (int k = 0; k < 16; k += 2) cap.of_any(s[k], s[k + 1]);
          }
        }
        const int row = g * 32 + (q & 1) * 16;
        const float4* const less = reinterpret_cast<const float4*>(rows.less + row);
        const float2 scale = make_float2(csc, csc);
        float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        if (!masked) {
#pragma unroll
          for (int k = 0; k < 16; k += 4) {
            const float4 l = less[k / 4];
            const float2 e0 = __ffma2_rn(make_float2(s[k], s[k + 1]), scale, make_float2(l.x, l.y)), e1 = __ffma2_rn(make_float2(s[k + 2], s[k + 3]), scale, make_float2(l.z, l.w));
            acc[0] = __fadd2_rn(acc[0], make_float2(tree_ex2(e0.x), tree_ex2(e0.y)));
            acc[1] = __fadd2_rn(acc[1], make_float2(tree_ex2(e1.x), tree_ex2(e1.y)));
          }
        } else {
          const int4* const sees = reinterpret_cast<const int4*>(rows.sees + row);
          const float2* const less2 = reinterpret_cast<const float2*>(less);
#pragma unroll
          for (int k = 0; k < 16; k += 2) {
            const int4 see = sees[k / 2];
            const float2 e = __ffma2_rn(make_float2(s[k], s[k + 1]), scale, less2[k / 2]);
            acc[(k / 2) & 1] = __fadd2_rn(acc[(k / 2) & 1], make_float2(key.x <= see.x && see.x < key.y && key.place > see.y ? tree_ex2(e.x) : 0.f,
                                                                         key.x <= see.z && see.z < key.y && key.place > see.w ? tree_ex2(e.y) : 0.f));
          }
        }
        sum += (acc[0].x + acc[1].x) + (acc[0].y + acc[1].y);
      };
      float s0[16], s1[16];
      if (note.tiles > 0) load(s0, 0);
#pragma unroll 1
      for (int i = 0; i < note.tiles; ++i) {
        const int4 bound = sm.rows[j % NR][i].bound[g];
        const bool any = __any_sync(0xffffffffu, key.x <= bound.y && key.y > bound.x && key.place > bound.z);
        const bool masked = !__all_sync(0xffffffffu, key.x <= bound.x && key.y > bound.y && key.place > bound.w);
        wait_on_16(s0);
        load(s1, 2 * i + 1);
        if (any) add(s0, 2 * i, masked);
        wait_on_16(s1);
        if (i + 1 < note.tiles) load(s0, 2 * i + 2);
        if (any) add(s1, 2 * i + 1, masked);
      }
      tc_fence_before();
      const bool last = note.flags & LAST;
      if (last && g > 0) { sm.sums[n % NU][g - 1][in] = sum; mbar_arrive(smem_u32(&sm.sums_full[n % NU])); }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(smem_u32(&sm.s_empty[j % NS]));
        mbar_arrive(smem_u32(&sm.r_empty[j % NR]));
        if (last) mbar_arrive(smem_u32(&sm.u_empty[n % NU]));
      }
      if (last && g == 0) {
        if (!wait(sm.sums_full[n % NU], n / NU)) return;
#pragma unroll
        for (int k = 0; k < KW_SETS - 1; ++k) sum += sm.sums[n % NU][k][in];
        if (chunks > 1) {                                    // behind the places of the weights
          parts[(long long)(units / chunks + part) * KT + in] = sum;
          if (part % chunks == 0) reinterpret_cast<int*>(parts)[(long long)(part / chunks) * KT + in] = key.at;
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
    for (int i = 0; i < NR; ++i) { mbar_init(smem_u32(&sm.r_full[i]), 1); mbar_init(smem_u32(&sm.r_empty[i]), KW_SUM); }
    for (int i = 0; i < NU; ++i) { mbar_init(smem_u32(&sm.sums_full[i]), KT * (KW_SETS - 1)); mbar_init(smem_u32(&sm.u_empty[i]), KW_SUM); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(smem_u32(&sm.tmem), NS * RT);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  asm volatile("griddepcontrol.wait;" ::: "memory");         // what the plan kernel writes
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  uint8_t* const space = static_cast<uint8_t*>(t.a.workspace);
  const Head head = *reinterpret_cast<const Head*>(space);
  const int units = (int)head.units * head.chunks;
  KwBlock<DH, CAP> block{t, map_q, map_k, sm, box, units, head.chunks, space, head.rows_at, reinterpret_cast<float*>(space + head.parts_at), sm.tmem};
  if (blockIdx.x < units) {
    if (warp == 0) block.produce();
    else if (warp == 1) { if (elect_one()) block.issue(); }
    else if (warp >= KW_FIRST) block.sum_up();
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
  const uint8_t* const space = static_cast<const uint8_t*>(t.a.workspace);
  const Head head = *reinterpret_cast<const Head*>(space);
  if (head.chunks == 1) return;
  const float* const parts = reinterpret_cast<const float*>(space + head.parts_at);
  const int* const at_of = reinterpret_cast<const int*>(parts);
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < head.units * KT; i += (long long)gridDim.x * 256) {
    const int at = at_of[i];
    if (at == -1) continue;
    const float* const part = parts + (head.units + i / KT * head.chunks) * KT + i % KT;
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
  PHX_CUDA_TRY(launch_programmatic(key_weights_tc_kernel<DH, CAP>, dim3(blocks), dim3(KW_THREADS), smem, stream, t, map_q, map_k, box), err);
  dispatch_note(DK_KEY_WEIGHTS_TC);
  return PHX_OK;
}
template <int DH>
phx_status launch(const WeightsView& t, const CUtensorMap& map_q, const CUtensorMap& map_k, int box, int blocks, cudaStream_t stream, std::string& err) {
  return t.a.cap_method == 0 ? launch<DH, 0>(t, map_q, map_k, box, blocks, stream, err) : t.a.cap_method == 1 ? launch<DH, 1>(t, map_q, map_k, box, blocks, stream, err)
                                                                                                               : launch<DH, 2>(t, map_q, map_k, box, blocks, stream, err);
}

// Tiles of rows that a call may have, whatever its offsets are, and what is written down about them; the most units of a request
long long row_tiles_bound(const WeightsView& t, int batch) { return ((long long)t.c.num_tokens / (HT / t.group) + batch) * t.c.num_kv_heads; }
long long units_bound(const WeightsView& t) { return ((long long)t.c.table_cols * t.c.page_size + KT - 1) / KT * t.c.num_kv_heads; }

}  // namespace

// Up to 16 rows a key head the mma.sync kernel reads the keys once, as fast as they come.  What is written down about rows (13 bytes each) and one request's keys has to fit three quarters of the
// workspace, some two million rows and 100 thousand tiles of keys; calls beyond that stay with it, too, as do those without new tokens, which have no queries to copy, and
// those without a column in their tables, which only have that to report.
bool weights_tc_supported(const WeightsView& t) {
  if (t.c.num_tokens == 0 || t.c.table_cols == 0 || t.group > HT || (long long)t.a.max_tokens * t.group <= 16) return false;
  return UNITS_AT + row_tiles_bound(t, t.c.batch < TREE_MAX_SPLIT_BATCH ? t.c.batch : TREE_MAX_SPLIT_BATCH) * (long long)sizeof(RowNote) + units_bound(t) * (long long)sizeof(UnitNote) <= t.a.workspace_bytes / 4 * 3;
}

phx_status weights_tc_launch(WeightsView& t, cudaStream_t stream, std::string& err) {
  t.rows = HT / t.group * t.group; t.keys = KT;
  int box = KT;                                    // the largest power of two that a page is a multiple of, at most a tile
  while (t.c.page_size % box != 0) box /= 2;
  CUtensorMap map_q, map_k;
  phx_status s = tree_query_map(&map_q, t, err);
  if (s == PHX_OK) s = tree_pool_map(&map_k, t, box, true, err);
  const WeightsView whole = t;
  const int per_tile = t.rows / t.group, sms = device_sms();
  // as many requests at a time as a block plans and whose notes fit
  const long long room = t.a.workspace_bytes - UNITS_AT - row_tiles_bound(t, t.c.batch < TREE_MAX_SPLIT_BATCH ? t.c.batch : TREE_MAX_SPLIT_BATCH) * (long long)sizeof(RowNote);
  const long long fit = room / (units_bound(t) * (long long)sizeof(UnitNote));
  const int slice = (int)(fit < TREE_MAX_SPLIT_BATCH ? fit : TREE_MAX_SPLIT_BATCH);
  for (int b0 = 0; s == PHX_OK && b0 < whole.c.batch; b0 += slice) {
    t = whole;
    t.c.batch = whole.c.batch - b0 < slice ? whole.c.batch - b0 : slice;
    t.c.q_start += b0; t.c.lengths += b0; t.c.block_table += b0 * t.c.table_stride;
    long long tiles = (t.a.max_keys + KT - 1) / KT;
    if (t.decay == 1.0f) {
      const long long seen = ((long long)t.sinks + KT - 1) / KT + ((long long)t.window + t.a.max_tokens + KT - 3) / KT + 1;
      if (seen < tiles) tiles = seen;
    }
    // Tiles of rows in chunks where units alone leave blocks idle in a last round: about six rounds then, of two pairs at least
    const long long units = tiles * t.c.num_kv_heads * t.c.batch, row_tiles = (t.a.max_tokens + per_tile - 1) / per_tile;
    t.chunks = 1;
    if (units < 4 * sms) {
      const long long pairs = (row_tiles + 1) / 2, want = (6ll * sms + units - 1) / units;
      long long per = pairs / want > 2 ? pairs / want : 2;   // pairs of a chunk
      if ((pairs + per - 1) / per > 15) per = (pairs + 14) / 15;
      t.chunks = (int)((pairs + per - 1) / per);
    }
    const long long notes = units * t.chunks + row_tiles * t.c.num_kv_heads * t.c.batch, plans = (notes + PLAN_THREADS / 32 - 1) / (PLAN_THREADS / 32);
    PHX_CUDA_TRY(launch_programmatic(key_weights_plan_kernel, dim3((unsigned)(plans < 4 * sms ? plans : 4 * sms)), dim3(PLAN_THREADS), 0, stream, t, box), err);
    const int blocks = (int)(units * t.chunks < sms ? units * t.chunks : sms);
    s = t.c.key_size == 32 ? launch<32>(t, map_q, map_k, box, blocks, stream, err) : t.c.key_size == 64 ? launch<64>(t, map_q, map_k, box, blocks, stream, err) : launch<128>(t, map_q, map_k, box, blocks, stream, err);
    if (s == PHX_OK && t.chunks > 1) {
      const long long joins = (units * KT + 255) / 256;
      const cudaError_t e = launch_programmatic(key_weights_join_kernel, dim3((unsigned)(joins < 4 * sms ? joins : 4 * sms)), dim3(256), 0, stream, t);
      if (e != cudaSuccess) { err = cudaGetErrorString(e); s = PHX_E_CUDA; }
    }
  }
  return s;
}

}  // namespace phx
