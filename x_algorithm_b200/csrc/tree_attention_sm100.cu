// Attention over a paged cache on Blackwell tensor cores (tcgen05 + TMEM + TMA), for requests of more than 16 query rows a key head; the
// semantics are tree_attention.cu's.  A block (192 threads, two on an SM) takes 128 rows - 128 / group tokens with the group's query heads - of one
// request and key head, or a stretch of its keys (TreePlan):
//   warp 0      TMA producer: the Q tile, then per tile of keys the K and the V rows, page by page (a box is what of a page lies in a tile)
//   warp 1      MMA issuer: S = Q K^T into tensor memory, later O += P V with P read from tensor memory and V as an MN-major operand
//   warps 2-5   softmax: thread = query row; S row from tensor memory, mask, exponentials and row sum in registers, P rounded to bf16 back over
//               the S columns, O rescaled there when the row's reference moved; at the end the row is normalised and stored, or left as a part
// New tokens' keys cost only the tiles that some row of the block sees: each tile's spans are compared with the rows' places first (neither, some or
// all of its keys seen by all), and only tiles of the second kind are masked.  Those are searched for infinities and NaN among the values as well, which
// 0 * V would spread to rows that do not see them: they are taken out of shared memory and added to the rows that do at the end.
// Waits are bounded; when one runs out the flag is raised and every later wait returns at once, so all roles drain.
#include <string.h>

#include "sm100_ptx.cuh"
#include "tree_attention.cuh"

namespace phx {
namespace {

using namespace sm100;

constexpr int QT = 128;                 // query rows of a block
constexpr int TC_THREADS = 192;
constexpr int SLAB = QT * 128;          // bytes of one [128 rows x 64 bf16] swizzled tile
constexpr int NEW_TILES = 2048;         // tiles of new keys that are classified; those behind count as seen in part
constexpr int KT = 64;                  // keys of a tile: S of two tiles and O share the block's 256 columns of tensor memory
// K and V buffers each: 64 KB a block
__host__ __device__ constexpr int tc_buffers(int dh) { return dh == 64 ? 4 : 2; }

__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
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

// Wait for the tensor-memory loads in flight.  The 32 registers are operands, so that no use of them is scheduled in front of it.
__device__ __forceinline__ void tmem_ld_wait_on(float* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]), "+f"(r[8]), "+f"(r[9]), "+f"(r[10]),
                 "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]), "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]),
                 "+f"(r[21]), "+f"(r[22]), "+f"(r[23]), "+f"(r[24]), "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]), "+f"(r[30]), "+f"(r[31])
               :: "memory");
}

template <int DH>
struct TcSmem {
  static constexpr int DCH = DH / 64, NB = tc_buffers(DH);
  uint8_t q[DCH * SLAB];
  uint8_t k[NB][DCH * KT * 128];
  uint8_t v[NB][DCH * KT * 128];
  int2 span[2][KT];                     // of a masked tile's keys
  uint32_t need[NEW_TILES / 32], mask[NEW_TILES / 32];
  uint64_t q_full, k_full[NB], k_empty[NB], v_full[NB], v_empty[NB], s_full[2], p_ready, o_done;
  uint32_t there[8];                    // which boxes of a tile lie in pages of the pool
  uint32_t tmem;
  int odd;                              // a masked tile of the piece held infinities or NaN
  TreePlan<TC_THREADS> plan;
};

// The tiles of a piece that are needed, one after the other; a role's own copy keeps the word of bits it is in
template <int DH>
struct TileWalk {
  const TcSmem<DH>* sm;
  int new0, last;                       // the first tile with new keys; behind the piece's last
  int at = -1;
  uint32_t need = 0, mask = 0;
  __device__ __forceinline__ void fetch(int i) {
    if ((i >> 5) != at) { at = i >> 5; need = sm->need[at]; mask = sm->mask[at]; }
  }
  // the first from `tile` on; `last`: none
  __device__ __forceinline__ int next(int tile) {
    while (tile < last) {
      const int i = tile - new0;
      if (i < 0 || i >= NEW_TILES) return tile;
      fetch(i);
      const uint32_t rest = need >> (i & 31);
      if (rest & 1) return tile;
      tile += rest ? __ffs(rest) - 1 : 32 - (i & 31);
    }
    return last;
  }
  // whether some of the block's rows do not see some of its keys (those of pages outside the pool and behind the last key aside)
  __device__ __forceinline__ bool masked(int tile) {
    const int i = tile - new0;
    if (i < 0) return false;
    if (i >= NEW_TILES) return true;
    fetch(i);
    return (mask >> (i & 31)) & 1;
  }
};

template <int DH, int CAP>
struct TcBlock {
  static constexpr int DCH = DH / 64, NB = tc_buffers(DH);
  static constexpr uint32_t BLK = DCH * KT * 128, TM_S = 0, TM_O = 128;
  const TreeView& t;
  const CUtensorMap& map_q;
  const CUtensorMap& map_kv;
  TcSmem<DH>& sm;
  int box;                                                 // rows of a K / V copy
  int seq = 0;                                             // tiles taken so far, over all pieces
  uint32_t q_phase = 0;

  __device__ void piece(const TreePiece& pc) {
    const int warp = warp_index(), lane = threadIdx.x & 31, group = t.group, tokens_per_tile = t.rows / group;
    const KeyRange kr = key_range(t.c, pc.b);
    const CacheRequest& rq = kr.rq;
    const int token0 = pc.row_tile * tokens_per_tile;
    volatile int* const verr = t.c.status_dev;
    if (threadIdx.x == 0) {
      sm.odd = 0;
      if (kr.keys < (long long)rq.cached + rq.tokens) cache_report(t.c, CACHE_BAD_PAGE);
    }
    const uint32_t tmem = sm.tmem;
    int first_page = -1;
    if (warp == 0) {                                        // on their way under what follows
      first_page = page_of(kr, pc.begin);
      if (elect_one()) {
        mbar_expect_tx(smem_u32(&sm.q_full), DCH * t.rows * 128);
        for (int c = 0; c < DCH; ++c) tma_load_3d(smem_u32(sm.q) + c * SLAB, &map_q, smem_u32(&sm.q_full), c * 64, pc.h * group, rq.row0 + token0);
      }
      __syncwarp();
    }

    // ---- which tiles of new keys the block's rows see ----------------------------------------------------------------
    const int new0 = rq.cached / KT, key_tiles = (kr.keys + KT - 1) / KT, last = min(pc.end, key_tiles);   // the first tile with new keys
    if (last > new0) {
      for (int i = threadIdx.x; i < NEW_TILES / 32; i += TC_THREADS) sm.need[i] = sm.mask[i] = 0;
      int lo = 0x7fffffff, hi = -1;
      for (int i = lane; i < tokens_per_tile && token0 + i < rq.tokens; i += 32) {
        const int pre = span_of(t, rq, token0 + i).x;
        if (pre >= 0) { lo = min(lo, pre); hi = max(hi, pre); }
      }
      lo = __reduce_min_sync(0xffffffffu, lo); hi = __reduce_max_sync(0xffffffffu, hi);
      __syncthreads();
      for (int tile = max(pc.begin, new0) + warp; tile < last && tile - new0 < NEW_TILES; tile += TC_THREADS / 32) {
        bool any = false, all = true;
#pragma unroll
        for (int i = 0; i < KT / 32; ++i) {
          const int key = tile * KT + i * 32 + lane;
          if (key >= kr.keys) { all = false; continue; }
          if (key < rq.cached) { any = true; continue; }
          const int2 s = span_of(t, rq, key - rq.cached);
          any |= s.x <= hi && s.y > lo;
          all &= s.x <= lo && s.y > hi;
        }
        any = __any_sync(0xffffffffu, any) && hi >= 0;
        all = __all_sync(0xffffffffu, all);
        if (lane == 0) {
          const int i = tile - new0;
          if (any) atomicOr(&sm.need[i >> 5], 1u << (i & 31));
          if (!all) atomicOr(&sm.mask[i >> 5], 1u << (i & 31));
        }
      }
    }
    __syncthreads();
    TileWalk<DH> walk{&sm, new0, last};
    const int first = walk.next(pc.begin);

    if (warp == 0) {
      produce(kr, pc, first, walk, first == pc.begin ? first_page : page_of(kr, first));
    } else if (warp == 1) {
      if (elect_one()) issue(first, walk, tmem);
    } else {
      softmax(kr, pc, token0, first, walk, tmem);
    }
    for (int tile = first; tile < last; tile = walk.next(tile + 1)) ++seq;
    q_phase ^= 1;
    tc_fence_before();
    __syncthreads();                                        // Q, the buffers and O are free for the next piece
    tc_fence_after();
  }

  // page of box `lane` of a tile, the last of which may lie behind the keys
  __device__ __forceinline__ int page_of(const KeyRange& kr, int tile) const {
    const int lane = threadIdx.x & 31;
    const long long key = (long long)tile * KT + lane * box;
    return lane < KT / box && key < kr.keys ? kr.table[(int)key / t.c.page_size] : -1;
  }
  __device__ __forceinline__ void produce(const KeyRange& kr, const TreePiece& pc, int first, TileWalk<DH> walk, int page) {
    const int last = walk.last;
    const int lane = threadIdx.x & 31, boxes = KT / box, v_off = t.c.num_kv_heads * t.c.page_size, no_row = (int)(2 * t.c.num_pages * v_off);
    volatile int* const verr = t.c.status_dev;
    // row of the pool of box `lane` of a tile
    auto row_of = [&](int tile, int page) {
      const int key = tile * KT + lane * box;
      return page >= 0 && page < t.c.num_pages ? (page * 2 * t.c.num_kv_heads + pc.h) * t.c.page_size + key % t.c.page_size : no_row;
    };
    int rows[4], before[4];                                // of this tile's boxes, of the tile's before
    int j = seq;
    // K runs a tile ahead of V: a buffer is free once S of the tile before in it has been computed
    for (int tile = first;; ++j) {
      const bool have = tile < last;
      const int after = have ? walk.next(tile + 1) : last, page_after = page_of(kr, after);
      if (have) {
        const int row = row_of(tile, page);
        const uint32_t there = __ballot_sync(0xffffffffu, row != no_row);
        if (lane < boxes && row == no_row && tile * KT + lane * box < kr.keys) cache_report(t.c, CACHE_BAD_PAGE);
#pragma unroll
        for (int p = 0; p < 4; ++p) rows[p] = __shfl_sync(0xffffffffu, row, p);
        if (elect_one()) {
          const int b = j % NB;
          mbar_wait(smem_u32(&sm.k_empty[b]), (uint32_t)((j / NB) & 1) ^ 1u, verr);
          sm.there[j & 7] = there;
          mbar_expect_tx(smem_u32(&sm.k_full[b]), BLK);
#pragma unroll
          for (int p = 0; p < 4; ++p)
            if (p < boxes)
              for (int c = 0; c < DCH; ++c) tma_load_2d(smem_u32(sm.k[b]) + c * KT * 128 + p * box * 128, &map_kv, smem_u32(&sm.k_full[b]), c * 64, rows[p]);
        }
      }
      if (j > seq && elect_one()) {
        const int i = j - 1, b = i % NB;
        mbar_wait(smem_u32(&sm.v_empty[b]), (uint32_t)((i / NB) & 1) ^ 1u, verr);
        mbar_expect_tx(smem_u32(&sm.v_full[b]), BLK);
#pragma unroll
        for (int p = 0; p < 4; ++p)
          if (p < boxes)
            for (int c = 0; c < DCH; ++c)
              tma_load_2d(smem_u32(sm.v[b]) + c * KT * 128 + p * box * 128, &map_kv, smem_u32(&sm.v_full[b]), c * 64, before[p] == no_row ? no_row : before[p] + v_off);
      }
      __syncwarp();
      if (!have) break;
#pragma unroll
      for (int p = 0; p < 4; ++p) before[p] = rows[p];
      tile = after; page = page_after;
    }
  }

  __device__ __forceinline__ void issue(int first, TileWalk<DH> walk, uint32_t tmem) {
    const int last = walk.last;
    constexpr uint32_t idesc_s = make_idesc(QT, KT), idesc_o = make_idesc_b_mn(QT, DH);
    volatile int* const verr = t.c.status_dev;
    auto issue_s = [&](int j) {                             // S(j) = Q K(j)^T into S buffer j & 1
      const int b = j % NB;
      mbar_wait(smem_u32(&sm.k_full[b]), (uint32_t)((j / NB) & 1), verr);
      tc_fence_after();
#pragma unroll
      for (int c = 0; c < DCH; ++c) {
        const uint64_t qd = make_smem_desc(smem_u32(sm.q) + c * SLAB), kd = make_smem_desc(smem_u32(sm.k[b]) + c * KT * 128);
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_bf16(tmem + TM_S + (j & 1) * KT, qd + (uint64_t)(k * 2), kd + (uint64_t)(k * 2), idesc_s, (c | k) != 0);
      }
      umma_commit(smem_u32(&sm.k_empty[b]));
      umma_commit(smem_u32(&sm.s_full[j & 1]));
    };
    mbar_wait(smem_u32(&sm.q_full), q_phase, verr);
    int ahead = first, j = seq, js = seq;                   // the next tile whose S is to be issued, its number
    auto issue_next = [&]() { if (ahead < last) { issue_s(js++); ahead = walk.next(ahead + 1); } };
    issue_next();
    for (; j < js; ++j) {
      issue_next();                                         // its S buffer was last read by the softmax whose P has been awaited below
      const int b = j % NB;
      mbar_wait(smem_u32(&sm.v_full[b]), (uint32_t)((j / NB) & 1), verr);
      mbar_wait(smem_u32(&sm.p_ready), (uint32_t)(j & 1), verr);
      tc_fence_after();
#pragma unroll
      for (int kk = 0; kk < KT / 16; ++kk) {
        const uint64_t vd = make_smem_desc_mn(smem_u32(sm.v[b]) + kk * 16 * 128, KT * 128, 1024);
        umma_ts(tmem + TM_O, tmem + TM_S + (j & 1) * KT + kk * 8, vd, idesc_o, (j - seq) | kk);
      }
      umma_commit(smem_u32(&sm.v_empty[b]));
      umma_commit(smem_u32(&sm.o_done));
    }
  }

  __device__ __forceinline__ void softmax(const KeyRange& kr, const TreePiece& pc, int token0, int first, TileWalk<DH> walk, uint32_t tmem) {
    const int last = walk.last;
    const int lane = threadIdx.x & 31, quad = warp_index() & 3, r = quad * 32 + lane, group = t.group;
    const CacheRequest& rq = kr.rq;
    volatile int* const verr = t.c.status_dev;
    const uint32_t lane_base = (uint32_t)(quad * 32) << 16;
    const int token = token0 + r / group;
    const bool valid = r < t.rows && token < rq.tokens;
    const int pre = valid ? span_of(t, rq, token).x : -1;
    const bool busy = __any_sync(0xffffffffu, valid);       // a warp without rows only keeps the others company
    const TreeCap cap(t);
    const float csc = CAP ? 1.0f : t.csc;
    float m = valid ? -INFINITY : 0.f, l = 0.f;
    int j = seq;

    const uint32_t all_there = (1u << (KT / box)) - 1;
    for (int tile = first; tile < last; ++j) {
      const uint32_t ph = (uint32_t)(j & 1), s_col = tmem + TM_S + (j & 1) * KT + lane_base;
      bool masked = walk.masked(tile) || (tile + 1) * KT > kr.keys;
      mbar_wait(smem_u32(&sm.s_full[j & 1]), (uint32_t)((j >> 1) & 1), verr);
      tc_fence_after();
      float s[KT];
      if (busy) {                                           // on its way under what follows
#pragma unroll
        for (int c = 0; c < KT / 32; ++c) tmem_ld32_nowait(s_col + c * 32, reinterpret_cast<uint32_t*>(s) + c * 32);
      }
      const uint32_t there = sm.there[j & 7];
      masked |= there != all_there;
      const int after = walk.next(tile + 1);
      if (masked) {                                         // the same for all 128 threads
        if (r < KT) {
          const int key = tile * KT + r;
          int2 s = make_int2(0, 0x7fffffff);                // cached: seen by all but padding
          if (key >= kr.keys || !((there >> (r / box)) & 1)) s = make_int2(0x7fffffff, -1);
          else if (key >= rq.cached) s = span_of(t, rq, key - rq.cached);
          sm.span[j & 1][r] = s;
        }
        // infinities and NaN among the values: out of the product
        mbar_wait(smem_u32(&sm.v_full[j % NB]), (uint32_t)((j / NB) & 1), verr);
        uint4* const v = reinterpret_cast<uint4*>(sm.v[j % NB]);
        bool odd = false;
        for (int i = r; i < (int)BLK / 16; i += 128) {
          uint4 x = v[i];
          if (odd_pair(x.x) || odd_pair(x.y) || odd_pair(x.z) || odd_pair(x.w)) {
            uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) { if (odd_value(w[k])) w[k] &= 0xffff0000u; if (odd_value(w[k] >> 16)) w[k] &= 0xffffu; }
            v[i] = make_uint4(w[0], w[1], w[2], w[3]);
            odd = true;
          }
        }
        if (odd) sm.odd = 1;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        softmax_sync();
      }
      float alpha = 1.0f;
      if (busy) {
        tmem_ld_wait_on(s);
        tmem_ld_wait_on(s + 32);
        bool small = false;
        if (CAP == 2) {                                      // tanh by its polynomial where all of the warp's logits are small against the cap
          float big = 0.f;
#pragma unroll
          for (int k = 0; k < KT; ++k) big = fmaxf(big, fabsf(s[k]));
          small = __all_sync(0xffffffffu, !valid || big * cap.small_scale <= TreeCap::SMALL);
        }
        if (CAP == 2 && small) {
#pragma unroll
          for (int k = 0; k < KT; k += 2) cap.of_small(s[k], s[k + 1]);
        } else if (CAP) {
#pragma unroll
          for (int k = 0; k < KT; ++k) s[k] = cap.template of<CAP>(s[k]);
        }
        if (masked) {
#pragma unroll
          for (int k = 0; k < KT; ++k) { const int2 sp = sm.span[j & 1][k]; if (!(sp.x <= pre && pre < sp.y)) s[k] = -INFINITY; }
        }
        float b4[4] = {s[0], s[1], s[2], s[3]};              // four chains of three-input max
#pragma unroll
        for (int k = 4; k + 7 < KT; k += 8) {
          b4[0] = max3(b4[0], s[k], s[k + 1]); b4[1] = max3(b4[1], s[k + 2], s[k + 3]);
          b4[2] = max3(b4[2], s[k + 4], s[k + 5]); b4[3] = max3(b4[3], s[k + 6], s[k + 7]);
        }
        float bm = fmaxf(max3(b4[0], b4[1], b4[2]), b4[3]);
#pragma unroll
        for (int k = KT - 4; k < KT; ++k) bm = fmaxf(bm, s[k]);   // the tail that the 8-wide loop leaves
        // The reference only has to bound the exponentials: it moves when the maximum has outgrown it by 2^8 (P stays below 256, as exact in bf16 as below
        // 1), which spares rescaling O for almost every tile.  Each row moves its own.
        const float m_true = fmaxf(m, bm * csc);
        const bool move = valid && (m_true > m + 8.0f || (m == -INFINITY && m_true != -INFINITY));
        const float m_new = move ? m_true : m, mns = m_new == -INFINITY ? 0.f : m_new;
        if (move) alpha = tree_ex2(m - mns);                 // -inf: 0
        m = m_new;
        if (j > seq && __any_sync(0xffffffffu, alpha != 1.0f)) {
          mbar_wait(smem_u32(&sm.o_done), ph ^ 1u, verr);    // O of the tiles before must be complete
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
            sum2[k & 1] = __fadd2_rn(sum2[k & 1], x);        // the sum keeps fp32
            pw[k] = pack_bf2(x.x, x.y);                      // rounded for the product
          }
          tmem_st16(s_col + c * 16, pw);
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        tc_fence_before();
        l = l * alpha + ((sum2[0].x + sum2[0].y) + (sum2[1].x + sum2[1].y));
      }
      // S of this tile did not wait for P V of the one before: its barrier must not run two phases ahead of the issuer
      if (j > seq) mbar_wait(smem_u32(&sm.o_done), ph ^ 1u, verr);
      mbar_arrive(smem_u32(&sm.p_ready));
      tile = after;
    }

    // ---- the row: normalised and stored, or left as a part ---------------------------------------------------------------
    const bool any = j > seq;
    if (any) {
      mbar_wait(smem_u32(&sm.o_done), (uint32_t)((j - 1) & 1), verr);
      tc_fence_after();
    } else {
      mbar_wait(smem_u32(&sm.q_full), q_phase, verr);        // no product has waited for Q: its copy must be over before the next one's
    }
    const bool none = l == 0.f || pre < 0;                   // no key seen, or a padding token
    const float inv = none ? 0.f : 1.0f / l;
    const int head = pc.h * group + r % group;
    const long long part_row = (long long)(2 * blockIdx.x + pc.part()) * t.rows + r;
    uint16_t* const out = t.a.out + ((long long)(rq.row0 + token) * t.a.num_q_heads + head) * DH;
    if (busy) {
#pragma unroll
      for (int c = 0; c < DH / 32; ++c) {
        float o[32];
        __syncwarp();
        if (any) {
          tmem_ld32(tmem + TM_O + lane_base + c * 32, reinterpret_cast<uint32_t*>(o));
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = 0.f;
        }
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
    }
    // what the row sees of the infinities and NaN that were taken out of the masked tiles, onto what has been stored
    if (sm.odd != 0 && valid && !none) {
#pragma unroll 1
      for (int tile = first; tile < last; tile = walk.next(tile + 1)) {
        bool masked = (tile + 1) * KT > kr.keys || walk.masked(tile);
        for (int key = tile * KT; key < min((tile + 1) * KT, kr.keys); key += box) masked |= (unsigned)kr.table[key / t.c.page_size] >= (unsigned)t.c.num_pages;
        if (!masked) continue;
#pragma unroll 1
        for (int key = tile * KT; key < min((tile + 1) * KT, kr.keys); ++key) {
          const int page = kr.table[key / t.c.page_size];
          const int2 s = key >= rq.cached ? span_of(t, rq, key - rq.cached) : make_int2(0, 0x7fffffff);
          if ((unsigned)page >= (unsigned)t.c.num_pages || !(s.x <= pre && pre < s.y)) continue;
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

template <int DH, int CAP>
__global__ void __launch_bounds__(TC_THREADS, 2) tree_tc_kernel(const __grid_constant__ TreeView t, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_kv, int box) {
  extern __shared__ uint8_t smem_bytes[];
  TcSmem<DH>& sm = *reinterpret_cast<TcSmem<DH>*>(smem_bytes + ((1024u - (smem_u32(smem_bytes) & 1023u)) & 1023u));
  const int warp = warp_index();
  if (threadIdx.x == 0) {
    *gave_up() = 0;
    prefetch_map(&map_q); prefetch_map(&map_kv);
    mbar_init(smem_u32(&sm.q_full), 1); mbar_init(smem_u32(&sm.p_ready), 128); mbar_init(smem_u32(&sm.o_done), 1);
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

  TcBlock<DH, CAP> block{t, map_q, map_kv, sm, box};
  if (t.split == 0) {
    const int b = blockIdx.z;
    const KeyRange kr = key_range(t.c, b);
    if (!kr.rq.ok && threadIdx.x == 0) cache_report(t.c, CACHE_BAD_OFFSETS);
    const int row_tiles = tree_row_tiles(t, kr.rq.tokens), tiles = tree_key_tiles(t, kr.keys);
    for (int rt = blockIdx.x; rt < row_tiles; rt += gridDim.x) block.piece(TreePiece{b, (int)blockIdx.y, rt, 0, tiles, tiles});
  } else {
    sm.plan.make(t);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (blockIdx.x == 0)
      for (int b = threadIdx.x; b < t.c.batch; b += TC_THREADS)
        if (!cache_request(t.c, b).ok) cache_report(t.c, CACHE_BAD_OFFSETS);
    const long long start = sm.plan.bound(blockIdx.x), end = sm.plan.bound(blockIdx.x + 1);
    if (threadIdx.x == 0) t.join[blockIdx.x].rows = 0;
    for (long long pos = start; pos < end;) {
      const bool first = pos == start;
      long long unit_end;
      const TreePiece pc = sm.plan.piece(t, pos, end, &pos, &unit_end);
      if (first && threadIdx.x == 0) sm.plan.note_join(t, blockIdx.x, pc, unit_end);
      if (pc.begin < pc.end) block.piece(pc);
    }
  }

  settle();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(sm.tmem, 256);
  }
}

// Queries as [token][head][column]; a box is 64 columns of the group's heads of as many tokens as 128 rows hold
phx_status query_map(CUtensorMap* map, const TreeView& t, std::string& err) {
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

template <int DH, int CAP>
phx_status launch(const TreeView& t, cudaStream_t stream, std::string& err) {
  constexpr int smem = (int)sizeof(TcSmem<DH>) + 1024;
  static_assert(2 * (smem + 1024 + 64) <= 228 * 1024, "two blocks share an SM");
  static SmemLimit limit;
  PHX_CUDA_TRY(limit.raise(tree_tc_kernel<DH, CAP>, smem), err);
  int box = KT;                                    // the largest power of two that a page is a multiple of, at most a tile
  while (t.c.page_size % box != 0) box /= 2;
  CUtensorMap map_q, map_kv;
  phx_status s = query_map(&map_q, t, err);
  if (s == PHX_OK) s = tree_pool_map(&map_kv, t, box, err);
  if (s != PHX_OK) return s;
  const long long row_tiles = ((long long)t.a.max_tokens * t.group + t.rows - 1) / t.rows;
  const dim3 grid = t.split ? dim3(t.split) : dim3((unsigned)(row_tiles < 65535 ? row_tiles : 65535), t.c.num_kv_heads, t.c.batch);
  tree_tc_kernel<DH, CAP><<<grid, TC_THREADS, smem, stream>>>(t, map_q, map_kv, box);
  PHX_CUDA_TRY(cudaGetLastError(), err);
  dispatch_note(DK_TREE_TC);
  return PHX_OK;
}
template <int DH>
phx_status launch(const TreeView& t, cudaStream_t stream, std::string& err) {
  if (t.a.cap_method == 0 && !(t.a.sm_scale > 0.f)) return launch<DH, 3>(t, stream, err);
  return t.a.cap_method == 0 ? launch<DH, 0>(t, stream, err) : t.a.cap_method == 1 ? launch<DH, 1>(t, stream, err) : launch<DH, 2>(t, stream, err);
}

}  // namespace

bool tree_tc_supported(const TreeView& t) { return (t.c.key_size == 64 || t.c.key_size == 128) && t.group <= QT; }
void tree_tc_shape(TreeView& t) { t.rows = QT / t.group * t.group; t.keys = KT; t.setup = 6; }
int tree_tc_blocks_per_sm() { return 2; }
phx_status tree_tc_launch(const TreeView& t, cudaStream_t stream, std::string& err) {
  return t.c.key_size == 64 ? launch<64>(t, stream, err) : launch<128>(t, stream, err);
}

}  // namespace phx
