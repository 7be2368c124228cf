// Attention over a paged cache on Blackwell tensor cores (tcgen05 + TMEM + TMA), for requests of more than 16 query rows a key head; the
// semantics are tree_attention.cu's.  A block (192 threads, two on an SM) takes 128 rows - 128 / group tokens with the group's query heads - of one
// request and key head after the other, or stretches of their keys (PieceWalk); its roles go through the same pieces, each at its own pace:
//   warp 0      TMA producer: the Q tile, then per tile of keys the K and the V rows, page by page (a box is what of a page lies in a tile), and a note
//               about the tile: which boxes lie in pages of the pool, whether some row does not see some key, whether it is the piece's last
//   warp 1      MMA issuer: S = Q K^T into tensor memory, a tile ahead, later O += P V with P read from tensor memory and V as an MN-major operand
//   warps 2-5   softmax: thread = query row; S row from tensor memory, mask, exponentials and row sum in registers, P rounded to bf16 back over
//               the S columns, O rescaled there when the row's reference moved; at the end the row is normalised and stored, or left as a part
// The next piece's Q and keys are on their way while a piece's rows are stored.  (With a barrier of the whole block between pieces, and the tiles of new
// keys classified in front of each, a piece of 16 tiles spent 9 of 31 us on that.)
// New tokens' keys cost only the tiles that some row of the block sees: the producer compares each such tile's spans with the rows' places (no key
// seen, some, or all of them by all rows), and only tiles of the second kind are masked.  Those are searched for infinities and NaN among the values as well, which
// 0 * V would spread to rows that do not see them: they are taken out of shared memory and added to the rows that do at the end.
// Waits are bounded; when one runs out the flag is raised, every later wait of any role fails at once, and a role whose wait failed is done.
// Measured: 8192 tokens that see themselves, 16 heads of 128, 506 us = 1086 TFLOP/s (bound by a tile's chain of load, maximum, exponentials and store, 1800
// cycles of two blocks in turns, and by the special-function unit, 1024 of them); 24 trees of 32 over up to 8192 keys, 32 heads of 128 (465 MB), 100 us = 4.6 TB/s,
// with capped logits 106; 74 such trees over 8192 keys each 405 us = 6.2 TB/s.
// With a window what a row sees of a masked tile is two words: of the cached keys, and of a chain's, a stretch and the first ones, worked out from four numbers; of new keys with
// spans what the producer has laid beside the tile's note.  No barrier of the softmax threads is needed then, and the values are searched by the issuer's warp while the softmax is at the
// logits.  Measured (us): 4 x 2048 tokens in a chain, window 1024, 16 heads on 4 of 128: 122; 24 trees of 32, windows of 4096, 32 heads on 8 of 128, capped: 109; 32 x 512 candidates, window 512, 8
// heads of 64: 82 - with the search by the softmax threads 120, 107, 88 (37 x 512 tokens in a chain, 8 heads of 64: 78, 75 by the issuer's warp); with spans compared key by key behind a barrier 152
// and 101 for the first and the third.  Divisions by a tile's keys in PieceWalk, which every role does for every unit, cost 6, 7 and 6 us.
// Heads of 32 (with a window) are tiles of 64 columns whose second half is zeros behind the tensors' edge; products take half the steps.
#include <string.h>

#include "sm100_ptx.cuh"
#include "tree_attention.cuh"

namespace phx {
namespace {

using namespace sm100;

constexpr int QT = 128;                 // query rows of a block
constexpr int TC_THREADS = 192;
constexpr int SLAB = QT * 128;          // bytes of one [128 rows x 64 bf16] swizzled tile
constexpr int KT = 64;                  // keys of a tile: S of two tiles and O share the block's 256 columns of tensor memory
// K and V buffers each: 64 KB a block
__host__ __device__ constexpr int tc_buffers(int dh) { return dh == 128 ? 2 : 4; }

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float min3(float a, float b, float c) {
  float d;
  asm("min.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// D[tmem] (+)= A[tmem] * B[smem desc]
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accum)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// what the producer notes about a tile
struct TileNote {
  int tile;
  uint32_t flags;                       // bits 0 .. 3: boxes in pages of the pool; MASKED, LAST of the piece, FINAL of the block; PLACES: new keys that some row's window leaves out
};
struct alignas(16) WindowNote : TileNote {
  int cached, keys;                     // of the request
};
template <class View> using NoteOf = std::conditional_t<has_window<View>, WindowNote, TileNote>;
constexpr uint32_t MASKED = 16, LAST = 32, FINAL = 64, PLACES = 128, BOXES = 15;

template <int DH, class View>
struct TcSmem {
  static constexpr int DCH = (DH + 63) / 64, NB = tc_buffers(DH);
  uint8_t q[DCH * SLAB];
  uint8_t k[NB][DCH * KT * 128];
  uint8_t v[NB][DCH * KT * 128];
  // (pre, end) of a masked tile's keys; with a window those of new keys alone, and their places, of as many tiles as notes
  int2 span[has_window<View> ? 8 : 2][KT];
  int place[has_window<View> ? 8 : 1][has_window<View> ? KT : 1];
  NoteOf<View> note[8];
  uint64_t q_full, q_empty, k_full[NB], k_empty[NB], v_full[NB], v_empty[NB], s_full[2], p_ready, o_done, o_empty, together;
  uint32_t tmem;
  int odd[2];                           // the last piece (by its number's parity) with infinities or NaN in a masked tile, plus 1
  TreePlan<TC_THREADS> plan;
};

// The pieces of a block, the same for every role: its stretch of the places, every gridDim.x-th unit, or the units of its place in the grid
template <int DH, class View>
struct PieceWalk {
  const View& t;
  const TcSmem<DH, View>& sm;
  long long pos, end;
  int row_tile;
  __device__ __forceinline__ PieceWalk(const View& view, const TcSmem<DH, View>& mem) : t(view), sm(mem), pos(0), end(0), row_tile(blockIdx.x) {
    if (t.split) { pos = sm.plan.bound(blockIdx.x); end = sm.plan.bound(blockIdx.x + 1); }
    else if (t.turns) { pos = blockIdx.x; end = sm.plan.all(t); }
  }
  __device__ __forceinline__ bool next(TreePiece* p) {
    if (t.split) {
      long long unit_end;
      while (pos < end) {
        *p = sm.plan.piece(t, pos, end, &pos, &unit_end);
        if (p->begin < p->end) return true;
      }
      return false;
    }
    if (t.turns) {
      if (pos >= end) return false;
      *p = sm.plan.unit(t, pos);
      pos += gridDim.x;
      return true;
    }
    const KeyRange k = key_range(t.c, blockIdx.z);
    if (row_tile >= tree_row_tiles(t, k.rq.tokens)) return false;
    const int tiles = unit_tiles(t, k);
    *p = TreePiece{(int)blockIdx.z, (int)blockIdx.y, row_tile, 0, tiles, tiles};
    row_tile += gridDim.x;
    return true;
  }
};

template <int DH, int CAP, class View>
struct TcBlock {
  static constexpr bool WINDOW = has_window<View>;
  static constexpr int DCH = (DH + 63) / 64, NB = tc_buffers(DH);
  static constexpr uint32_t BLK = DCH * KT * 128, TM_S = 0, TM_O = 128;
  const View& t;
  const CUtensorMap& map_q;
  const CUtensorMap& map_kv;
  TcSmem<DH, View>& sm;
  int box;                                                 // rows of a K / V copy
  uint32_t tmem;

  __device__ __forceinline__ bool wait(const uint64_t& bar, int phase) const { return mbar_wait(smem_u32(&bar), (uint32_t)(phase & 1), t.c.status_dev); }
  // ---- TMA producer (a whole warp; one lane issues) ----------------------------------------------------------------------
  // Its chain of instructions for a tile has to be shorter than the tile's softmax, beside whose warps it issues: pages and spans are asked for a tile
  // ahead, by loads without a condition (a value chosen between a load and a constant waits for the load), and places in pages are counted on, not divided.
  // (8192 tokens that see themselves, 16 heads of 128: 716 us before the first, 577 before the second, 502 then.)
  __device__ __forceinline__ void produce(PieceWalk<DH, View> walk) {
    const int lane = threadIdx.x & 31, boxes = KT / box, page_size = t.c.page_size, v_off = t.c.num_kv_heads * page_size, page_rows = 2 * v_off;
    const int no_row = (int)(t.c.num_pages * page_rows), tokens_per_tile = rows_tokens(t), cols_on = KT / page_size, slots_on = KT % page_size;
    TreePiece pc, after;
    bool more = walk.next(&after);
    int j = 0;                                              // tiles of the block so far
    for (int piece = 0; more; ++piece) {
      pc = after;
      const KeyRange kr = key_range(t.c, pc.b);
      const CacheRequest& rq = kr.rq;
      const int keys = kr.keys, token0 = pc.row_tile * tokens_per_tile, last_col = keys > 0 ? (keys - 1) / page_size : 0;
      int begin = pc.begin, last = min(pc.end, (keys + KT - 1) / KT);
      // with a window: the tiles of the rows, and the places behind which the least and the last of the rows' windows begin
      TileRange range{0, 0, 0};
      int behind_least = 0, behind_last = 0;
      if constexpr (WINDOW) {
        const int token1 = min(token0 + tokens_per_tile, rq.tokens) - 1;
        range = tile_range(t, kr, token0, token1);
        begin = range.at(pc.begin);
        last = min(min(range.at(pc.end - 1) + 1, (keys + KT - 1) / KT), range.end);
        if (t.positions) {
          int least = 0x7fffffff, most = 0;
          for (int i = token0 + lane; i <= token1; i += 32) { const int p = place_of(t, rq, i); least = min(least, p); most = max(most, p); }
          behind_least = (int)__reduce_min_sync(0xffffffffu, least) - t.window; behind_last = (int)__reduce_max_sync(0xffffffffu, most) - t.window;
        } else {
          behind_least = place_of(t, rq, token0) - t.window; behind_last = place_of(t, rq, token1) - t.window;
        }
      }
      const int old_tiles = min(rq.cached, keys) / KT, head_row = pc.h * page_size;   // tiles in front of the first with new keys
      if (lane == 0 && keys < (long long)rq.cached + rq.tokens) cache_report(t.c, CACHE_BAD_PAGE);
      // box `lane` of the tile that is looked up: column of the table, place in the page, page
      int col, slot, page;
      auto look_up = [&](int tile) { const int key = tile * KT + lane * box; col = key / page_size; slot = key - col * page_size; };
      auto ask_page = [&]() { page = keys > 0 ? kr.table[min(col, last_col)] : -1; };
      look_up(begin);
      ask_page();
      auto queries = [&]() {
        if (piece > 0 && !wait(sm.q_empty, piece - 1)) return false;
        __syncwarp();
        if (elect_one()) {
          mbar_expect_tx(smem_u32(&sm.q_full), DCH * t.rows * 128);
          for (int c = 0; c < DCH; ++c) tma_load_3d(smem_u32(sm.q) + c * SLAB, &map_q, smem_u32(&sm.q_full), c * 64, pc.h * t.group, rq.row0 + token0);
        }
        __syncwarp();
        return true;
      };
      // With four buffers the producer is here before the last S of the piece before has been multiplied, and looks things up first: 37 x 512 tokens, 8 heads, window 64, 42.5 -> 41.2 us; with two
      // buffers it is late, and Q goes first (128 columns 58.6, 60.3 the other way).
      constexpr bool Q_LATE = WINDOW && NB > 2;
      if (!Q_LATE && !queries()) return;
      // the places that the block's rows take, once a tile of new keys asks for them
      int lo = 0x7fffffff, hi = -2;
      auto places = [&]() {
        hi = -1;
        for (int i = lane; i < tokens_per_tile && token0 + i < rq.tokens; i += 32) {
          const int pre = span_of(t, rq, token0 + i).x;
          if (pre >= 0) { lo = min(lo, pre); hi = max(hi, pre); }
        }
        lo = __reduce_min_sync(0xffffffffu, lo); hi = __reduce_max_sync(0xffffffffu, hi);
      };
      int2 spans[KT / 32];                                   // of this lane's keys of tile spans_of
      int spans_of = -1;
      auto ask_spans = [&](int tile) {
        spans_of = tile;
#pragma unroll
        for (int i = 0; i < KT / 32; ++i) spans[i] = span_of(t, rq, max(0, min(tile * KT + i * 32 + lane - rq.cached, rq.tokens - 1)));
      };
      // the first tile from `tile` on of which some row sees some key (`last`: none); *masked: not every row every key
      auto next_tile = [&](int tile, bool* masked) {
        for (; tile < last; ++tile) {
          if constexpr (WINDOW) {
            if (tile >= range.sinks && tile < range.first) tile = range.first;
            if (tile >= last) break;
          }
          *masked = false;
          if (tile < old_tiles) {
            if constexpr (WINDOW) *masked = tile * KT <= behind_last && (tile + 1) * KT > t.sinks;
            return tile;
          }
          if (hi == -2) places();
          if (spans_of != tile) ask_spans(tile);
          bool any = false, all = true;
#pragma unroll
          for (int i = 0; i < KT / 32; ++i) {
            const int key = tile * KT + i * 32 + lane;
            const bool there = key < keys, cached = key < rq.cached;
            bool some = there, every = there;
            if constexpr (WINDOW) {
              const int place = there ? key_place(t, rq, key) : 0;
              some &= place > behind_least; every &= place > behind_last;
            }
            any |= some && (cached || (spans[i].x <= hi && spans[i].y > lo));
            all &= every && (cached || (spans[i].x <= lo && spans[i].y > hi));
          }
          ask_spans(tile + 1);
          any = __any_sync(0xffffffffu, any) && hi >= 0;
          *masked = !__all_sync(0xffffffffu, all);
          if (any) return tile;
        }
        return last;
      };
      bool masked = false, masked_next = false;
      int tile = next_tile(begin, &masked);
      if (tile >= last) { tile = begin; masked = true; }     // a piece that no row sees anything of is one masked tile all the same
      if (tile != begin) { look_up(tile); ask_page(); }
      more = walk.next(&after);
      int before[4] = {no_row, no_row, no_row, no_row};      // rows of the pool of the boxes of the tile whose V is still to be asked for
      auto values = [&](int i) {
        if (!wait(sm.v_empty[i % NB], i / NB - 1)) return false;   // its buffer is free once the tile before in it has been multiplied (the first wait passes)
        __syncwarp();
        if (elect_one()) {
          const int b = i % NB;
          mbar_expect_tx(smem_u32(&sm.v_full[b]), BLK);
#pragma unroll
          for (int p = 0; p < 4; ++p)
            if (p < boxes)
              for (int c = 0; c < DCH; ++c)
                tma_load_2d(smem_u32(sm.v[b]) + c * KT * 128 + p * box * 128, &map_kv, smem_u32(&sm.v_full[b]), c * 64, before[p] == no_row ? no_row : before[p] + v_off);
        }
        __syncwarp();
        return true;
      };
      if (Q_LATE && !queries()) return;
      for (int first = j;; ++j) {                            // K runs a tile ahead of V
        bool in_keys = lane < boxes && tile * KT + lane * box < keys;
        // a box that no row's window reaches and no first key lies in: its page may be another request's by now
        if constexpr (WINDOW) in_keys &= tile * KT + (lane + 1) * box - 1 > min(behind_least, rq.cached - 1) || tile * KT + lane * box < t.sinks;
        const bool ok = in_keys && (unsigned)page < (unsigned)t.c.num_pages;
        const int row = ok ? page * page_rows + head_row + slot : no_row;
        const uint32_t there = __ballot_sync(0xffffffffu, ok);
        if (in_keys && !ok) cache_report(t.c, CACHE_BAD_PAGE);
        int rows[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) rows[p] = __shfl_sync(0xffffffffu, row, p);
        if (!wait(sm.k_empty[j % NB], j / NB - 1)) return;
        bool places = false;
        if constexpr (WINDOW) {
          const bool is_chain_call = is_chain(t);                             // what the softmax asks for of new keys, before the next tile's are asked for
          if ((masked || there != (1u << boxes) - 1) && !is_chain_call && tile >= old_tiles) {
#pragma unroll
            for (int i = 0; i < KT / 32; ++i) {
              const int key = tile * KT + i * 32 + lane;
              const bool fresh = key >= rq.cached && key < keys;
              sm.span[j & 7][i * 32 + lane] = fresh ? span_of(t, rq, key - rq.cached) : make_int2(0x7fffffff, -1);
              const int place = fresh ? key_place(t, rq, key) : 0x7fffffff;
              if (t.positions) sm.place[j & 7][i * 32 + lane] = place;
              places |= place <= behind_last;
            }
            places = __any_sync(0xffffffffu, places);
          }
        }
        const int follows = next_tile(tile + 1, &masked_next);
        __syncwarp();
        if (elect_one()) {
          const int b = j % NB;
          NoteOf<View> n;
          n.tile = tile;
          if constexpr (WINDOW) { n.cached = rq.cached; n.keys = keys; }
          n.flags = there | (masked || there != (1u << boxes) - 1 ? MASKED : 0u) | (follows >= last ? LAST | (more ? 0u : FINAL) : 0u) | (places ? PLACES : 0u);
          sm.note[j & 7] = n;                              // in front of the arrival, which publishes it
          mbar_expect_tx(smem_u32(&sm.k_full[b]), BLK);
#pragma unroll
          for (int p = 0; p < 4; ++p)
            if (p < boxes)
              for (int c = 0; c < DCH; ++c) tma_load_2d(smem_u32(sm.k[b]) + c * KT * 128 + p * box * 128, &map_kv, smem_u32(&sm.k_full[b]), c * 64, rows[p]);
        }
        __syncwarp();
        if (follows == tile + 1) {
          slot += slots_on; col += cols_on;
          if (slot >= page_size) { slot -= page_size; ++col; }
        } else {
          look_up(follows);
        }
        ask_page();
        if (j > first && !values(j - 1)) return;
#pragma unroll
        for (int p = 0; p < 4; ++p) before[p] = rows[p];
        if (follows >= last) break;
        tile = follows; masked = masked_next;
      }
      if (!values(j++)) return;
    }
  }

  // Infinities and NaN among a masked tile's values: out of the product.  By THREADS threads, of which this is number `r`; piece: what sm.odd notes
  template <int THREADS> __device__ __forceinline__ void take_out_odd(int buffer, int r, int piece) const {
    uint4* const v = reinterpret_cast<uint4*>(sm.v[buffer]);
    bool odd = false;
    for (int i = r; i < (int)BLK / 16; i += THREADS) {
      uint4 x = v[i];
      if (odd_pair(x.x) || odd_pair(x.y) || odd_pair(x.z) || odd_pair(x.w)) {
        uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) { if (odd_value(w[k])) w[k] &= 0xffff0000u; if (odd_value(w[k] >> 16)) w[k] &= 0xffffu; }
        v[i] = make_uint4(w[0], w[1], w[2], w[3]);
        odd = true;
      }
    }
    if (odd) sm.odd[piece & 1] = piece + 1;
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  // The same by a warp, which looks first whether there is one: 0 x + 0 is NaN then
  __device__ __forceinline__ void look_for_odd(int buffer, int piece) const {
    const uint4* const v = reinterpret_cast<const uint4*>(sm.v[buffer]);
    const int lane = threadIdx.x & 31;
    const __nv_bfloat162 zero = __float2bfloat162_rn(0.f);
    __nv_bfloat162 sum[4] = {zero, zero, zero, zero};
#pragma unroll 8
    for (int i = 0; i < (int)BLK / 512; ++i) {
      const uint4 x = v[i * 32 + lane];
      const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) sum[k] = __hfma2(zero, *reinterpret_cast<const __nv_bfloat162*>(&w[k]), sum[k]);
    }
    sum[0] = __hadd2(__hadd2(sum[0], sum[1]), __hadd2(sum[2], sum[3]));
    if (__any_sync(0xffffffffu, odd_pair(*reinterpret_cast<const uint32_t*>(&sum[0])))) take_out_odd<32>(buffer, lane, piece);
    __syncwarp();
  }

  // ---- MMA issuer (one thread; with a window a warp, which searches masked tiles' values while the softmax is at their logits) ---
  __device__ __forceinline__ void issue() {
    const bool leader = !WINDOW || elect_one();
    auto wait = [&](const uint64_t& bar, int phase) { const bool there = this->wait(bar, phase); return WINDOW ? __all_sync(0xffffffffu, there) != 0 : there; };
    constexpr uint32_t idesc_s = make_idesc(QT, KT), idesc_o = make_idesc_b_mn(QT, DCH * 64);
    int s_pieces = 0;                                       // pieces whose S has been begun
    bool s_first = true;
    uint32_t flags_next = 0;
    auto issue_s = [&](int j) {                             // S(j) = Q K(j)^T into S buffer j & 1
      const int b = j % NB;
      if (s_first) { if (!wait(sm.q_full, s_pieces)) return false; ++s_pieces; }
      if (!wait(sm.k_full[b], j / NB)) return false;
      tc_fence_after();
      flags_next = sm.note[j & 7].flags;
      s_first = flags_next & LAST;
      if (!leader) return true;
#pragma unroll
      for (int c = 0; c < DCH; ++c) {
        const uint64_t qd = make_smem_desc(smem_u32(sm.q) + c * SLAB), kd = make_smem_desc(smem_u32(sm.k[b]) + c * KT * 128);
#pragma unroll
        for (int k = 0; k < (DH < 64 ? DH / 16 : 4); ++k) umma_bf16(tmem + TM_S + (j & 1) * KT, qd + (uint64_t)(k * 2), kd + (uint64_t)(k * 2), idesc_s, (c | k) != 0);
      }
      umma_commit(smem_u32(&sm.k_empty[b]));
      umma_commit(smem_u32(&sm.s_full[j & 1]));
      if (s_first) umma_commit(smem_u32(&sm.q_empty));
      return true;
    };
    if (!issue_s(0)) return;
    int pieces = 0;
    bool first = true;
    for (int j = 0;; ++j) {
      const uint32_t flags = flags_next;
      // the S buffer of the next tile was last read by the softmax whose P has been awaited below
      if (!(flags & FINAL) && !issue_s(j + 1)) return;
      const int b = j % NB;
      if (!wait(sm.v_full[b], j / NB)) return;
      if constexpr (WINDOW) { if (flags & MASKED) look_for_odd(b, pieces); }
      if (!wait(sm.p_ready, j)) return;
      if (WINDOW && (flags & LAST) && leader) mbar_arrive(smem_u32(&sm.together));   // sm.odd has its piece's answer (the softmax is done with that of the piece before)
      if (first && pieces > 0 && !wait(sm.o_empty, pieces - 1)) return;   // the rows of the piece before have been read
      tc_fence_after();
      if (leader) {
#pragma unroll
        for (int kk = 0; kk < KT / 16; ++kk) {
          const uint64_t vd = make_smem_desc_mn(smem_u32(sm.v[b]) + kk * 16 * 128, KT * 128, 1024);
          umma_ts(tmem + TM_O, tmem + TM_S + (j & 1) * KT + kk * 8, vd, idesc_o, !first || kk != 0);
        }
        umma_commit(smem_u32(&sm.v_empty[b]));
        umma_commit(smem_u32(&sm.o_done));
      }
      first = flags & LAST;
      pieces += first;
      if (flags & FINAL) return;
    }
  }

  // Which keys of a masked tile the row at `pre` sees, whose window begins behind place `behind`: of the cached ones and of a chain a stretch and the
  // first keys, in a few instructions; of new ones with spans those whose span has it, and those of their places that some window leaves out compared, too.
  __device__ __forceinline__ void window_seen(const WindowNote& note, bool all_there, int at, int pre, int behind, uint32_t* seen) const {
    const int key0 = note.tile * KT, cached = note.cached - key0;
    const bool chain = is_chain(t);                          // `pre` is a token's number then, and it sees up to itself
    auto below = [](int n) { uint32_t m; asm("bmsk.clamp.b32 %0, 0, %1;" : "=r"(m) : "r"(max(n, 0))); return m; };   // the lowest n bits
    const int end = min(note.keys - key0, chain ? cached + pre + 1 : cached), begin = behind + 1 - key0, first = t.sinks - key0;
#pragma unroll
    for (int w = 0; w < KT / 32; ++w) seen[w] = below(end - 32 * w) & (~below(begin - 32 * w) | below(first - 32 * w));
    if (!chain && cached < KT) {
#pragma unroll 1
      for (int k = 0; k < KT; k += 16) {                    // short code: it runs seldom, and is fetched anew each time
        uint32_t some = 0;
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const int4 s = *reinterpret_cast<const int4*>(&sm.span[at][k + i]);
          if (s.x <= pre && pre < s.y) some |= 1u << i;
          if (s.z <= pre && pre < s.w) some |= 2u << i;
        }
        some <<= k & 31;
        if (k < 32) seen[0] |= some; else seen[1] |= some;
      }
      if (note.flags & PLACES) {
#pragma unroll 1
        for (int k = max(0, cached); k < KT; ++k)
          if (sm.place[at][k] <= behind) { if (k < 32) seen[0] &= ~(1u << k); else seen[1] &= ~(1u << (k - 32)); }
      }
    }
    if (!all_there) {                                       // keys in no page of the pool
#pragma unroll 1
      for (int p = 0; p < KT / box; ++p)
        if (!((note.flags >> p) & 1))
          for (int k = p * box; k < (p + 1) * box; k += 16) { if (k < 32) seen[0] &= ~(0xffffu << k); else seen[1] &= ~(0xffffu << (k - 32)); }
    }
    if (pre < 0) seen[0] = seen[1] = 0;
  }

  // The polynomial and the exponential form of tanh differ in their last bits, so a key that a row does not see must not choose between them.  In a masked tile a row
  // goes by the logits that it sees, 16 keys at a time, in tensor memory and in a loop of its own: beside the code for whole tiles, where a warp takes one form
  // for all, such choices made that code 3 to 20 % slower (registers).  24 trees of 32 over up to 8192 keys, 32 heads of 128: 106 us, 152 with logits around the cap; 110 and 151 when
  // masked tiles were capped there by the warp's choice; 32 x 512 candidates under a cap 97 and 132, were 111 and 128.
  __device__ __forceinline__ void cap_masked(const TreeCap& cap, uint32_t s_col, const int2* span, int pre, const uint32_t* all_seen) const {
    tmem_ld_wait();
#pragma unroll 1
    for (int c = 0; c < KT / 16; ++c) {
      float x[16];
      tmem_ld16_nowait(s_col + c * 16, reinterpret_cast<uint32_t*>(x));
      tmem_ld_wait();
      uint32_t seen = 0;
      float most = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        bool see;
        if constexpr (WINDOW) { see = ((c < 2 ? all_seen[0] : all_seen[1]) >> ((c & 1) * 16 + k)) & 1; } else { const int2 sp = span[c * 16 + k]; see = sp.x <= pre && pre < sp.y; }
        if (see) { seen |= 1u << k; most = fmaxf(most, fabsf(x[k])); }
      }
      if (most * cap.small_scale <= TreeCap::SMALL) {
        if (seen != 0) {
#pragma unroll
          for (int k = 0; k < 16; k += 2) cap.of_small(x[k], x[k + 1]);
        }
      } else {
#pragma unroll
        for (int k = 0; k < 16; ++k) x[k] = cap.template of<2>(x[k]);
      }
      __syncwarp();
#pragma unroll
      for (int k = 0; k < 16; ++k) if (!((seen >> k) & 1)) x[k] = -INFINITY;
      tmem_st16(s_col + c * 16, reinterpret_cast<uint32_t*>(x));
    }
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
  }

  // ---- softmax (128 threads, one a row) ------------------------------------------------------------------------------------
  __device__ __forceinline__ void softmax(PieceWalk<DH, View> walk) {
    const int lane = threadIdx.x & 31, quad = warp_index() & 3, r = quad * 32 + lane, group = t.group;
    const uint32_t lane_base = (uint32_t)(quad * 32) << 16, all_there = (1u << (KT / box)) - 1;
    const TreeCap cap(t);
    const float csc = CAP ? 1.0f : t.csc;
    const int in_token = r % group, token_of = r / group;
    TreePiece pc, after;
    bool more = walk.next(&after);
    // this row of the piece to come: its request, token, place in the walk
    KeyRange kr_after;
    int pre_after = -1, behind_after = 0;
    bool valid_after = false;
    auto look = [&]() {
      kr_after = key_range(t.c, after.b);
      const int token = after.row_tile * rows_tokens(t) + token_of;
      valid_after = r < t.rows && token < kr_after.rq.tokens;
      pre_after = valid_after ? span_of(t, kr_after.rq, token).x : -1;
      if constexpr (WINDOW) behind_after = valid_after ? place_of(t, kr_after.rq, token) - t.window : 0;
    };
    if (more) look();
    int j = 0, together = 0;
    for (int piece = 0; more; ++piece) {
      pc = after;
      const KeyRange kr = kr_after;
      const CacheRequest& rq = kr.rq;
      const int pre = pre_after, behind = behind_after, token = pc.row_tile * rows_tokens(t) + token_of;
      const bool valid = valid_after, busy = __any_sync(0xffffffffu, valid);   // a warp without rows only keeps the others company
      float m = valid ? -INFINITY : 0.f, l = 0.f;
      const int first = j;
      for (;; ++j) {
        const uint32_t s_col = tmem + TM_S + (j & 1) * KT + lane_base;
        if (!wait(sm.s_full[j & 1], j >> 1)) return;
        tc_fence_after();
        float s[KT];
        if (busy) {                                         // on its way under what follows
#pragma unroll
          for (int c = 0; c < KT / 32; ++c) tmem_ld32_nowait(s_col + c * 32, reinterpret_cast<uint32_t*>(s) + c * 32);
        }
        const NoteOf<View> note = sm.note[j & 7];
        const bool masked = note.flags & MASKED;
        if (!WINDOW && masked) {                            // the same for all 128 threads
          if (r < KT) {
            const int key = note.tile * KT + r;
            int2 sp = make_int2(0, 0x7fffffff);             // cached: seen by all but padding
            if (key >= kr.keys || !((note.flags >> (r / box)) & 1)) sp = make_int2(0x7fffffff, -1);
            else if (key >= rq.cached) sp = span_of(t, rq, key - rq.cached);
            sm.span[j & 1][r] = sp;
          }
          if (!wait(sm.v_full[j % NB], j / NB)) return;
          take_out_odd<128>(j % NB, r, piece);
          mbar_arrive(smem_u32(&sm.together));              // a barrier of the softmax threads whose wait is bounded, too
          if (!wait(sm.together, together++)) return;
        }
        uint32_t seen[KT / 32] = {0, 0};
        if constexpr (WINDOW) {
          if (masked) { window_seen(note, (note.flags & BOXES) == all_there, j & 7, pre, behind, seen); __syncwarp(); }
        }
        float alpha = 1.0f;
        if (busy) {
          if (CAP == 2 && masked) {
            cap_masked(cap, s_col, sm.span[j & 1], pre, seen);
#pragma unroll
            for (int c = 0; c < KT / 32; ++c) tmem_ld32_nowait(s_col + c * 32, reinterpret_cast<uint32_t*>(s) + c * 32);
          }
          tmem_ld_wait_on(s);
          tmem_ld_wait_on(s + 32);
          // Four chains of three-input max.  tanh is monotone: without a mask one of the raw maximum serves for the row, and with the raw minimum it says
          // whether all of the warp's logits are small enough against the cap for its polynomial (but a padding token's, whose query has no part in others' rows).
          float bm;
          auto top_of = [&]() {
            float b4[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int k = 4; k + 7 < KT; k += 8) {
              b4[0] = max3(b4[0], s[k], s[k + 1]); b4[1] = max3(b4[1], s[k + 2], s[k + 3]);
              b4[2] = max3(b4[2], s[k + 4], s[k + 5]); b4[3] = max3(b4[3], s[k + 6], s[k + 7]);
            }
            return max3(fmaxf(b4[0], b4[1]), max3(b4[2], b4[3], s[KT - 4]), max3(s[KT - 3], s[KT - 2], s[KT - 1]));   // and the tail that the loop leaves
          };
          if (CAP == 2 && !masked) {
            float low[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
            for (int k = 4; k + 7 < KT; k += 8) {
              low[0] = min3(low[0], s[k], s[k + 1]); low[1] = min3(low[1], s[k + 2], s[k + 3]);
              low[2] = min3(low[2], s[k + 4], s[k + 5]); low[3] = min3(low[3], s[k + 6], s[k + 7]);
            }
            float least = min3(fminf(low[0], low[1]), min3(low[2], low[3], s[KT - 4]), min3(s[KT - 3], s[KT - 2], s[KT - 1]));
            bm = top_of();
            const bool small = __all_sync(0xffffffffu, pre < 0 || fmaxf(fabsf(bm), fabsf(least)) * cap.small_scale <= TreeCap::SMALL);
            if (cap.scale < 0.f) bm = least;                 // a negative scale turns the order round
            if (small) {
              cap.of_small(bm, least);
#pragma unroll
              for (int k = 0; k < KT; k += 2) cap.of_small(s[k], s[k + 1]);
            } else {
              bm = cap.template of<2>(bm);
#pragma unroll
              for (int k = 0; k < KT; ++k) s[k] = cap.template of<2>(s[k]);
            }
          } else if (CAP && CAP != 2) {
#pragma unroll
            for (int k = 0; k < KT; ++k) s[k] = cap.template of<CAP>(s[k]);
          }
          if (masked && CAP != 2) {
#pragma unroll
            for (int k = 0; k < KT; ++k) {
              if constexpr (WINDOW) { if (!((seen[k / 32] >> (k & 31)) & 1)) s[k] = -INFINITY; }
              else { const int2 sp = sm.span[j & 1][k]; if (!(sp.x <= pre && pre < sp.y)) s[k] = -INFINITY; }
            }
          }
          if (CAP != 2 || masked) bm = top_of();
          // The reference only has to bound the exponentials: it moves when the maximum has outgrown it by 2^8 (P stays below 256, as exact in bf16 as below
          // 1), which spares rescaling O for almost every tile.  Each row moves its own.
          const float m_true = fmaxf(m, bm * csc);
          const bool move = valid && (m_true > m + 8.0f || (m == -INFINITY && m_true != -INFINITY));
          const float m_new = move ? m_true : m, mns = m_new == -INFINITY ? 0.f : m_new;
          if (move) alpha = tree_ex2(m - mns);               // -inf: 0
          m = m_new;
          if (j > first && __any_sync(0xffffffffu, alpha != 1.0f)) {
            if (!wait(sm.o_done, j - 1)) return;             // O of the tiles before must be complete
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < DH / 16; ++c) {
              uint32_t o[16];
              tmem_ld16_nowait(tmem + TM_O + lane_base + c * 16, o);
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * alpha);
              tmem_st16(tmem + TM_O + lane_base + c * 16, o);
            }
          }
          const float2 c2 = make_float2(csc, csc), n2 = make_float2(-mns, -mns);
          float2 sum2[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
          for (int c = 0; c < KT / 32; ++c) {
            uint32_t pw[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const float2 e = __ffma2_rn(make_float2(s[c * 32 + 2 * k], s[c * 32 + 2 * k + 1]), c2, n2);
              const float2 x = make_float2(tree_ex2(e.x), tree_ex2(e.y));   // masked: 2^-inf = 0
              sum2[k & 1] = __fadd2_rn(sum2[k & 1], x);      // the sum keeps fp32
              pw[k] = pack_bf2(x.x, x.y);                    // rounded to bf16, which the product with bf16 values takes: outputs are 0.0020-0.0023 from 64 bits, 0.0017 of it their own rounding
            }
            tmem_st16(s_col + c * 16, pw);
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          tc_fence_before();
          l = l * alpha + ((sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y));
        }
        // S of this tile did not wait for P V of the one before: its barrier must not run two phases ahead of the issuer
        if (j > first && !wait(sm.o_done, j - 1)) return;
        mbar_arrive(smem_u32(&sm.p_ready));
        if (note.flags & LAST) break;
      }
      more = walk.next(&after);
      if (more) look();                                     // on its way under the row's end

      // ---- the row: normalised and stored, or left as a part -------------------------------------------------------------
      if (!wait(sm.o_done, j)) return;
      tc_fence_after();
      ++j;
      const bool none = l == 0.f || pre < 0;                 // no key seen, or a padding token
      const float inv = none ? 0.f : 1.0f / l;
      const int head = pc.h * group + in_token;
      const long long part_row = (long long)(2 * blockIdx.x + pc.part()) * t.rows + r;
      uint16_t* const out = t.a.out + ((long long)(rq.row0 + token) * t.a.num_q_heads + head) * DH;
      if (busy) {
#pragma unroll
        for (int c = 0; c < DH / 32; ++c) {
          float o[32];
          __syncwarp();
          tmem_ld32(tmem + TM_O + lane_base + c * 32, reinterpret_cast<uint32_t*>(o));
          if (c == DH / 32 - 1) { tc_fence_before(); mbar_arrive(smem_u32(&sm.o_empty)); }   // O may be begun anew
          if (valid && !pc.whole()) {
#pragma unroll
            for (int k = 0; k < 8; ++k) *reinterpret_cast<float4*>(t.part_o + part_row * DH + c * 32 + k * 4) = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
          } else if (valid) {
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = none ? 0.f : o[k] * inv;
#pragma unroll
            for (int k = 0; k < 4; ++k)
              *reinterpret_cast<uint4*>(out + c * 32 + k * 8) = make_uint4(pack_bf2(o[8 * k], o[8 * k + 1]), pack_bf2(o[8 * k + 2], o[8 * k + 3]),
                                                                           pack_bf2(o[8 * k + 4], o[8 * k + 5]), pack_bf2(o[8 * k + 6], o[8 * k + 7]));
          }
        }
        if (valid && !pc.whole()) t.part_ml[part_row] = none ? make_float2(-INFINITY, 0.f) : make_float2(m, l);
        if constexpr (WINDOW) { if (valid && pc.whole()) t.lse[(long long)(rq.row0 + token) * t.a.num_q_heads + head] = none ? -INFINITY : (m + log2f(l)) * TREE_LN2; }
      } else {
        mbar_arrive(smem_u32(&sm.o_empty));
      }
      // What the row sees of the infinities and NaN that were taken out of masked tiles, onto what has been stored.  (One of an unmasked tile is in there
      // already: adding it again changes nothing.)
      if constexpr (WINDOW) { if (!wait(sm.together, piece)) return; }
      if (sm.odd[piece & 1] == piece + 1 && valid && !none) {
        TileRange range{0, 0, 0};
        if constexpr (WINDOW) range = tile_range(t, kr, pc.row_tile * (t.rows / group), min((pc.row_tile + 1) * (t.rows / group), rq.tokens) - 1);
        const long long end = WINDOW ? pc.end * (long long)KT : min((long long)pc.end * KT, (long long)kr.keys);
#pragma unroll 1
        for (long long i = pc.begin * (long long)KT; i < end; ++i) {
          int key = (int)i;
          if constexpr (WINDOW) {
            const long long at = (long long)range.at((int)(i / KT)) * KT + i % KT;
            if (at >= kr.keys) break;
            key = (int)at;
            if (key_place(t, rq, key) <= behind) continue;
          }
          const int page = kr.table[key / t.c.page_size];
          const int2 sp = key >= rq.cached ? span_of(t, rq, key - rq.cached) : make_int2(0, 0x7fffffff);
          if ((unsigned)page >= (unsigned)t.c.num_pages || !(sp.x <= pre && pre < sp.y)) continue;
          const uint16_t* const v = t.c.pages + cache_row0(t.c, page, 1, pc.h) + (long long)(key % t.c.page_size) * DH;
#pragma unroll 1
          for (int d = 0; d < DH; ++d) {
            if (!odd_value(v[d])) continue;
            const float x = __uint_as_float((uint32_t)v[d] << 16);
            if (!pc.whole()) t.part_o[part_row * DH + d] += x;
            else { const bf16 y = f2bf(__uint_as_float((uint32_t)out[d] << 16) + x); out[d] = *reinterpret_cast<const uint16_t*>(&y); }
          }
        }
      }
    }
  }
};

template <int DH, int CAP, class View>
__global__ void __launch_bounds__(TC_THREADS, 2) tree_tc_kernel(const __grid_constant__ View t, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_kv, int box) {
  extern __shared__ uint8_t smem_bytes[];
  TcSmem<DH, View>& sm = *reinterpret_cast<TcSmem<DH, View>*>(smem_bytes + ((1024u - (smem_u32(smem_bytes) & 1023u)) & 1023u));
  const int warp = warp_index();
  if (threadIdx.x == 0) {
    *gave_up() = 0;
    sm.odd[0] = sm.odd[1] = 0;
    prefetch_map(&map_q); prefetch_map(&map_kv);
    mbar_init(smem_u32(&sm.q_full), 1); mbar_init(smem_u32(&sm.q_empty), 1); mbar_init(smem_u32(&sm.p_ready), 128); mbar_init(smem_u32(&sm.o_done), 1);
    mbar_init(smem_u32(&sm.o_empty), 128); mbar_init(smem_u32(&sm.together), has_window<View> ? 1 : 128);
    for (int i = 0; i < tc_buffers(DH); ++i) {
      mbar_init(smem_u32(&sm.k_full[i]), 1); mbar_init(smem_u32(&sm.k_empty[i]), 1);
      mbar_init(smem_u32(&sm.v_full[i]), 1); mbar_init(smem_u32(&sm.v_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) mbar_init(smem_u32(&sm.s_full[i]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(smem_u32(&sm.tmem), 256);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();

  if (t.split || t.turns) sm.plan.make(t);
  if (t.split) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
      t.join[blockIdx.x].rows = 0;
      const long long start = sm.plan.bound(blockIdx.x);
      if (start < sm.plan.bound(blockIdx.x + 1)) {
        long long next, unit_end;
        const TreePiece pc = sm.plan.piece(t, start, sm.plan.bound(blockIdx.x + 1), &next, &unit_end);
        sm.plan.note_join(t, blockIdx.x, pc, unit_end);
      }
    }
  }
  if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0)
    for (int b = threadIdx.x; b < t.c.batch; b += TC_THREADS)
      if (!cache_request(t.c, b).ok) cache_report(t.c, CACHE_BAD_OFFSETS);

  TcBlock<DH, CAP, View> block{t, map_q, map_kv, sm, box, sm.tmem};
  const PieceWalk<DH, View> walk(t, sm);
  if (warp == 0) {
    block.produce(walk);
  } else if (warp == 1) {
    PieceWalk<DH, View> mine = walk;
    TreePiece pc;
    if (mine.next(&pc) && (has_window<View> || elect_one())) block.issue();
  } else {
    block.softmax(walk);
  }

  settle();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(sm.tmem, 256);
  }
}

template <int DH, int CAP, class View>
phx_status launch(const View& t, cudaStream_t stream, std::string& err) {
  constexpr int smem = (int)sizeof(TcSmem<DH, View>) + 1024;
  static_assert(2 * (smem + 1024 + 64) <= 228 * 1024, "two blocks share an SM");
  static SmemLimit limit;
  PHX_CUDA_TRY(limit.raise(tree_tc_kernel<DH, CAP, View>, smem), err);
  int box = KT;                                    // the largest power of two that a page is a multiple of, at most a tile
  while (t.c.page_size % box != 0) box /= 2;
  CUtensorMap map_q, map_kv;
  phx_status s = tree_query_map(&map_q, t, err);
  if (s == PHX_OK) s = tree_pool_map(&map_kv, t, box, true, err);
  if (s != PHX_OK) return s;
  const long long row_tiles = ((long long)t.a.max_tokens * t.group + t.rows - 1) / t.rows;
  const dim3 grid = t.split || t.turns ? dim3(t.split ? t.split : t.turns) : dim3((unsigned)(row_tiles < 65535 ? row_tiles : 65535), t.c.num_kv_heads, t.c.batch);
  tree_tc_kernel<DH, CAP, View><<<grid, TC_THREADS, smem, stream>>>(t, map_q, map_kv, box);
  PHX_CUDA_TRY(cudaGetLastError(), err);
  dispatch_note(DK_TREE_TC);
  return PHX_OK;
}
template <class View>
phx_status launch_any(const View& t, cudaStream_t stream, std::string& err) {
  auto of = [&](auto dh) {
    constexpr int DH = decltype(dh)::value;
    if (t.a.cap_method == 0 && !(t.a.sm_scale > 0.f)) return launch<DH, 3>(t, stream, err);
    return t.a.cap_method == 0 ? launch<DH, 0>(t, stream, err) : t.a.cap_method == 1 ? launch<DH, 1>(t, stream, err) : launch<DH, 2>(t, stream, err);
  };
  if constexpr (has_window<View>) { if (t.c.key_size == 32) return of(std::integral_constant<int, 32>()); }
  return t.c.key_size == 64 ? of(std::integral_constant<int, 64>()) : of(std::integral_constant<int, 128>());
}

}  // namespace

// Queries as [token][head][column]; a box is 64 columns (behind a head of 32: zeros) of the group's heads of as many tokens as 128 rows hold
phx_status tree_query_map(CUtensorMap* map, const TreeView& t, std::string& err) {
  EncodeTiledFn fn = get_encode_fn(err);
  if (!fn) return PHX_E_CUDA;
  const cuuint64_t dh = (cuuint64_t)t.c.key_size;
  cuuint64_t dims[3] = {dh, (cuuint64_t)t.a.num_q_heads, (cuuint64_t)t.c.num_tokens};
  cuuint64_t strides[2] = {dh * 2, (cuuint64_t)t.a.q_stride * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)t.group, (cuuint32_t)(t.rows / t.group)}, estr[3] = {1, 1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<uint16_t*>(t.a.q), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) { err = "cuTensorMapEncodeTiled (queries) failed with code " + std::to_string((int)r); return PHX_E_CUDA; }
  return PHX_OK;
}

bool tree_tc_supported(const TreeView& t) { return (t.c.key_size == 64 || t.c.key_size == 128) && t.group <= QT; }
bool tree_tc_supported(const WindowView& t) { return t.group <= QT; }
void tree_tc_shape(TreeView& t) { t.rows = QT / t.group * t.group; t.keys = KT; t.setup = 6; }
int tree_tc_blocks_per_sm() { return 2; }
phx_status tree_tc_launch(const TreeView& t, cudaStream_t stream, std::string& err) { return launch_any(t, stream, err); }
phx_status tree_tc_launch(const WindowView& t, cudaStream_t stream, std::string& err) { return launch_any(t, stream, err); }

}  // namespace phx
