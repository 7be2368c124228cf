// Attention of a request's new tokens over its paged cache, their own keys included (phx_tree_attention_device):
//
//   o_i = sum_j p_ij v_j,   p_ij = softmax over the keys j that i sees of cap(q_i . k_j * scale)
//
// i sees every key cached before, and of the new tokens' keys those with pre[j] <= pre[i] < end[j].  The g query heads that share
// a key head are rows of one product: row r of a request and key head is token r / g, head r % g of the group, so K and V are read
// once for all of them.
//
// The mma.sync kernel, for requests of up to 16 such rows: a block's four warps share the rows and take 16 keys each in turn, every warp with
// its own ring of key and value tiles (copied by TMA, which swizzles them for ldmatrix; no barrier between the warps), running maximum, sum and
// output; they are joined once at the end.  Masked logits
// become -inf before the maximum; a value row that some of the tile's rows do not see must not reach them as 0 * NaN either, so tiles that are
// not seen whole are searched for infinities and NaN, which are then added to the rows that do see them, one by one.
// Bound by memory: 16 operations a byte of the cache, padded rows counted.  96 single tokens over up to 4096 keys, 4 key heads of 128 (382 MB), take 75 us = 5.1 TB/s, 138 us =
// 5.8 TB/s where all have 4096.  Two stages a warp and three blocks an SM against three and two: 75 / 78 us for the first, 138 / 137 for the second, 89 / 104 for
// 400 tokens over up to 1000 keys.
#include <math.h>

#include <string>
#include <vector>

#include "sm100_ptx.cuh"
#include "tree_attention.cuh"

namespace phx {
namespace {

constexpr int TREE_WARPS = 4;
constexpr int ROWS = 16;         // query rows of a tile
constexpr int KEYS = 16;         // keys of a warp's tile; a page holds whole tiles
constexpr int STAGES = 2;
constexpr int WIDE_CAP = 4;      // tanh under a cap so large that 1e-7 of it counts: small logits by the polynomial
using namespace sm100;

__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// byte of 16-byte piece `piece` of row `row` in a tile as TMA leaves it: 64 columns at a time, rows of 128 (64) bytes with their pieces exchanged
template <int DH>
__device__ __forceinline__ uint32_t tile_at(int row, int piece) {
  if (DH == 32) return (uint32_t)(row * 64 + ((piece ^ ((row >> 1) & 3)) << 4));
  return (uint32_t)(((piece >> 3) * KEYS + row) * 128 + (((piece & 7) ^ (row & 7)) << 4));
}

template <int DH>
struct TreeSmem {
  uint8_t kv[TREE_WARPS][STAGES][2][KEYS * DH * 2];
  uint64_t full[TREE_WARPS][STAGES];
  int tile[TREE_WARPS][STAGES];    // -1: no more
  int there[TREE_WARPS][STAGES];   // its keys sit in a page of the pool
  float m[TREE_WARPS][ROWS], l[TREE_WARPS][ROWS];
  TreePlan<32 * TREE_WARPS> plan;
};

template <int DH, int CAP>
__device__ __forceinline__ void tree_mma_piece(const TreeView& t, const CUtensorMap& map, TreeSmem<DH>& sm, const TreePiece& pc, int& seq) {
  constexpr int PIECES = DH / 8, KSTEPS = DH / 16, NT = DH / 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = pc.h, b = pc.b, group = t.group;
  const KeyRange kr = key_range(t.c, b);
  const CacheRequest& rq = kr.rq;
  const long long rows = (long long)rq.tokens * group, r0 = (long long)pc.row_tile * ROWS;
  const int n_tiles = min((kr.keys + KEYS - 1) / KEYS, pc.end * TREE_WARPS);
  if (threadIdx.x == 0 && kr.keys < (long long)rq.cached + rq.tokens) cache_report(t.c, CACHE_BAD_PAGE);
  const int v_off = t.c.num_kv_heads * t.c.page_size;                         // rows of the pool from a key to its value
  const int no_row = (int)(2 * t.c.num_pages * v_off);                        // behind the pool: zeros
  const uint32_t kv_smem = (uint32_t)__cvta_generic_to_shared(sm.kv[warp]);
  const TreeCap cap(t);

  {
    // rows lane / 4 and lane / 4 + 8 of the tile: token, its place in the walk, A fragments of the query
    int pre[2];
    const uint16_t* qrow[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const long long r = min(r0 + lane / 4 + 8 * i, rows - 1);
      const int tok = (int)(r / group), head = h * group + (int)(r - (long long)tok * group);
      pre[i] = span_of(t, rq, tok).x;
      qrow[i] = t.a.q + (long long)(rq.row0 + tok) * t.a.q_stride + head * DH;
    }
    int lo = 0, hi = -2;                               // the places that the tile's rows take in the walk, once they are asked for
    int next = pc.begin * TREE_WARPS + warp;           // the next tile of this warp that may be needed
    int ahead = -1, ahead_page = 0;                    // a tile whose page has been looked up
    auto page_of = [&](int tile) { return kr.table[tile * KEYS / t.c.page_size]; };
    auto load = [&](int at) {                          // the copy of the next tile that is needed into stage `at`, or a note that there is none
      int tile = -1;
      for (; next < n_tiles; next += TREE_WARPS) {
        if ((next + 1) * KEYS <= rq.cached) { tile = next; break; }
        if (hi == -2) {
          lo = min(pre[0] < 0 ? 0x7fffffff : pre[0], pre[1] < 0 ? 0x7fffffff : pre[1]);
          hi = max(pre[0], pre[1]);
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) { lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o)); hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o)); }
        }
        const int key = next * KEYS + (lane & (KEYS - 1)), j = key - rq.cached;   // this lane's key, among the new ones if j >= 0
        bool seen = key < kr.keys && hi >= 0;
        if (seen && j >= 0) { const int2 s = span_of(t, rq, j); seen = s.x <= hi && s.y > lo; }
        if (__any_sync(0xffffffffu, seen)) { tile = next; break; }
      }
      if (tile >= 0) {
        const int key = tile * KEYS, page = tile == ahead ? ahead_page : page_of(tile);
        const bool ok = page >= 0 && page < t.c.num_pages;
        const int row = ok ? (page * 2 * t.c.num_kv_heads + h) * t.c.page_size + key % t.c.page_size : no_row;
        __syncwarp();                                  // the stage's last reads are done
        if (elect_one()) {
          const uint32_t bar = smem_u32(&sm.full[warp][at]), dst = kv_smem + at * (2 * KEYS * DH * 2);
          mbar_expect_tx(bar, 2 * KEYS * DH * 2);
#pragma unroll
          for (int c = 0; c < (DH + 63) / 64; ++c) {
            tma_load_2d(dst + c * KEYS * 128, &map, bar, c * 64, row);
            tma_load_2d(dst + KEYS * DH * 2 + c * KEYS * 128, &map, bar, c * 64, ok ? row + v_off : no_row);
          }
        }
        if (lane == 0) {
          sm.there[warp][at] = ok;
          if (!ok) cache_report(t.c, CACHE_BAD_PAGE);
        }
        next += TREE_WARPS;
        ahead = next;
        if (ahead < n_tiles) ahead_page = page_of(ahead);
      }
      if (lane == 0) sm.tile[warp][at] = tile;
    };
    const int seq0 = seq;                              // tiles that this warp has taken so far, over all pieces: stage and parity of the next
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) load((seq0 + s) % STAGES);
    uint32_t q[KSTEPS][4];
#pragma unroll
    for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        q[k][i] = *reinterpret_cast<const uint32_t*>(qrow[i & 1] + k * 16 + (i >> 1) * 8 + (lane & 3) * 2);

    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    for (;; ++seq) {
      const int stage = seq % STAGES;
      load((seq + STAGES - 1) % STAGES);
      __syncwarp();
      const int tile = sm.tile[warp][stage], there = sm.there[warp][stage];
      if (tile < 0) break;
      mbar_wait(smem_u32(&sm.full[warp][stage]), (uint32_t)((seq / STAGES) & 1), t.c.status_dev);
      const uint32_t sk = kv_smem + stage * (2 * KEYS * DH * 2), sv = sk + KEYS * DH * 2;

      float s[KEYS / 8][4];
#pragma unroll
      for (int n = 0; n < KEYS / 8; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
        for (int n = 0; n < KEYS / 16; ++n) {          // 16 keys: two 8-key blocks, both halves of the 16 columns
          uint32_t kf[4];
          ldsm4(kf, sk + tile_at<DH>(n * 16 + (lane >> 4) * 8 + (lane & 7), k * 2 + ((lane >> 3) & 1)));
          mma_16816(s[2 * n], q[k], kf[0], kf[1]);
          mma_16816(s[2 * n + 1], q[k], kf[2], kf[3]);
        }

      // seen by every row: cached keys in pages of the pool
      const int key0 = tile * KEYS;
      const bool whole = key0 + KEYS <= min(rq.cached, kr.keys) && there;
      uint32_t seen[2] = {0xffu, 0xffu};               // bit 2 n + c: key 8 n + (lane & 3) * 2 + c, for either row
      if (CAP == WIDE_CAP) {
        float most = 0.f;
#pragma unroll
        for (int n = 0; n < KEYS / 8; ++n) most = fmaxf(fmaxf(fmaxf(most, fabsf(s[n][0])), fmaxf(fabsf(s[n][1]), fabsf(s[n][2]))), fabsf(s[n][3]));
        const bool small = __all_sync(0xffffffffu, most * cap.small_scale <= TreeCap::SMALL);
#pragma unroll
        for (int n = 0; n < KEYS / 8; ++n)
#pragma unroll
          for (int c = 0; c < 4; c += 2) {
            if (small) cap.of_small(s[n][c], s[n][c + 1]);
            else cap.of_any(s[n][c], s[n][c + 1]);           // the same bits for those that are small
          }
      } else {
#pragma unroll
        for (int n = 0; n < KEYS / 8; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float v = s[n][c];
            s[n][c] = CAP == 0 ? v * t.csc : cap.of<CAP>(v);
          }
      }
      if (!whole) {
        seen[0] = seen[1] = 0;
#pragma unroll
        for (int n = 0; n < KEYS / 8; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int in = n * 8 + (lane & 3) * 2 + c, key = key0 + in;
            const bool ok = key < kr.keys && there;
            int2 span = make_int2(0, 0x7fffffff);      // cached: seen by all
            if (ok && key >= rq.cached) span = span_of(t, rq, key - rq.cached);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const bool see = ok && span.x <= pre[i] && pre[i] < span.y;
              seen[i] |= see ? 1u << (2 * n + c) : 0u;
              if (!see) s[n][2 * i + c] = -INFINITY;
            }
          }
      }

      // running maximum, sum and output
      uint32_t p[KEYS / 16][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float mx = -INFINITY;
#pragma unroll
        for (int n = 0; n < KEYS / 8; ++n) mx = fmaxf(mx, fmaxf(s[n][2 * i], s[n][2 * i + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m[i], mx), base = mn == -INFINITY ? 0.f : mn, alpha = tree_ex2(m[i] - base);
        m[i] = mn;
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < KEYS / 8; ++n) {
          const float e0 = tree_ex2(s[n][2 * i] - base), e1 = tree_ex2(s[n][2 * i + 1] - base);
          sum += e0 + e1;
          p[n >> 1][(n & 1) * 2 + i] = pack_bf2(e0, e1);   // rounded to bf16 for the product with bf16 values; the sum keeps fp32
        }
        l[i] = l[i] * alpha + sum;
        if (__any_sync(0xffffffffu, alpha != 1.0f)) {
#pragma unroll
          for (int n = 0; n < NT; ++n) { acc[n][2 * i] *= alpha; acc[n][2 * i + 1] *= alpha; }
        }
      }
      if (!whole) {
        // infinities and NaN among the values: out of the product, and to the rows that see them
        bool odd = false;
#pragma unroll
        for (int i = 0; i < KEYS * PIECES / 32; ++i) {
          uint4 v;
          const uint32_t at = sv + (uint32_t)(i * 32 + lane) * 16;
          asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
          odd |= odd_pair(v.x) | odd_pair(v.y) | odd_pair(v.z) | odd_pair(v.w);
        }
        if (__any_sync(0xffffffffu, odd)) {
          for (int in = 0; in < KEYS; ++in) {
            // which of this thread's two rows see the key: the bits are with the quad's thread that holds the key's logit
            const int holder = (lane & ~3) | ((in & 7) >> 1);
            const uint32_t w0 = __shfl_sync(0xffffffffu, seen[0], holder), w1 = __shfl_sync(0xffffffffu, seen[1], holder);
            const int bit = 2 * (in >> 3) + (in & 1);
            const bool see[2] = {((w0 >> bit) & 1) != 0, ((w1 >> bit) & 1) != 0};
            for (int d = 0; d < NT; ++d)
              for (int c = 0; c < 2; ++c) {
                const uint32_t at = sv + tile_at<DH>(in, d) + ((lane & 3) * 2 + c) * 2;
                uint16_t v;
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at) : "memory");
                if (odd_value(v)) {
                  const float f = __uint_as_float((uint32_t)v << 16);
#pragma unroll
                  for (int dd = 0; dd < NT; ++dd)
                    if (dd == d) {
                      if (see[0]) acc[dd][c] += f;
                      if (see[1]) acc[dd][2 + c] += f;
                    }
                }
              }
          }
          __syncwarp();
          for (int i = 0; i < KEYS * PIECES / 32; ++i) {
            const uint32_t at = sv + (uint32_t)(i * 32 + lane) * 16;
            uint32_t v[4];
            asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(at) : "memory");
            for (int k = 0; k < 4; ++k) {
              if (odd_value(v[k])) v[k] &= 0xffff0000u;
              if (odd_value(v[k] >> 16)) v[k] &= 0xffffu;
            }
            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // a later tile is copied over these stores
          __syncwarp();
        }
      }
#pragma unroll
      for (int n = 0; n < KEYS / 16; ++n)
#pragma unroll
        for (int d = 0; d < DH / 16; ++d) {
          uint32_t vf[4];
          ldsm4_trans(vf, sv + tile_at<DH>(n * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), d * 2 + (lane >> 4)));
          mma_16816(acc[2 * d], p[n], vf[0], vf[1]);
          mma_16816(acc[2 * d + 1], p[n], vf[2], vf[3]);
        }
      __syncwarp();
    }

    // the warps' parts, joined: rows of DH floats over the tiles' memory
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
      if ((lane & 3) == 0) { sm.m[warp][lane / 4 + 8 * i] = m[i]; sm.l[warp][lane / 4 + 8 * i] = l[i]; }
    }
    __syncthreads();
    float* const part = reinterpret_cast<float*>(sm.kv);           // [warp][row][DH]
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        *reinterpret_cast<float2*>(part + ((warp * ROWS + lane / 4 + 8 * i) * DH + n * 8 + (lane & 3) * 2)) = make_float2(acc[n][2 * i], acc[n][2 * i + 1]);
    __syncthreads();
    for (int i = threadIdx.x; i < ROWS * PIECES; i += 32 * TREE_WARPS) {
      const int row = i / PIECES, piece = i % PIECES;
      if (r0 + row >= rows) continue;
      float top = sm.m[0][row];
#pragma unroll
      for (int w = 1; w < TREE_WARPS; ++w) top = fmaxf(top, sm.m[w][row]);
      const float base = top == -INFINITY ? 0.f : top;
      float sum = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < TREE_WARPS; ++w) {
        const float f = tree_ex2(sm.m[w][row] - base);
        if (sm.l[w][row] == 0.f) continue;                         // a part that saw no key
        sum += sm.l[w][row] * f;
        const float* src = part + (w * ROWS + row) * DH + piece * 8;
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] += src[k] * f;
      }
      const long long r = r0 + row;
      const int tk = (int)(r / group), head = h * group + (int)(r % group);
      const bool padding = span_of(t, rq, tk).x < 0;
      if (!pc.whole()) {                                           // the rest of the row's keys is another block's
        const long long at = (long long)(2 * blockIdx.x + pc.part()) * ROWS + row;
        *reinterpret_cast<float4*>(t.part_o + at * DH + piece * 8) = make_float4(o[0], o[1], o[2], o[3]);
        *reinterpret_cast<float4*>(t.part_o + at * DH + piece * 8 + 4) = make_float4(o[4], o[5], o[6], o[7]);
        if (piece == 0) t.part_ml[at] = padding ? make_float2(-INFINITY, 0.f) : make_float2(top, sum);
        continue;
      }
      const bool none = sum == 0.f || padding;                     // no key seen, or a padding token
      const float inv = none ? 0.f : 1.0f / sum;
#pragma unroll
      for (int k = 0; k < 8; ++k) o[k] = none ? 0.f : o[k] * inv;
      const uint4 v = make_uint4(pack_bf2(o[0], o[1]), pack_bf2(o[2], o[3]), pack_bf2(o[4], o[5]), pack_bf2(o[6], o[7]));
      *reinterpret_cast<uint4*>(t.a.out + ((long long)(rq.row0 + tk) * t.a.num_q_heads + head) * DH + piece * 8) = v;
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the next piece's tiles are copied over this
    __syncthreads();
  }
}

// blocks that share an SM: by shared memory (72 KB of tiles at key_size 128), and as many registers
template <int DH> constexpr int mma_blocks() { return DH == 128 ? 3 : 4; }

template <int DH, int CAP>
__global__ void __launch_bounds__(32 * TREE_WARPS, mma_blocks<DH>()) tree_mma_kernel(const TreeView t, const __grid_constant__ CUtensorMap map) {
  extern __shared__ uint8_t smem_bytes[];
  TreeSmem<DH>& sm = *reinterpret_cast<TreeSmem<DH>*>(smem_bytes + ((1024u - (smem_u32(smem_bytes) & 1023u)) & 1023u));
  if (threadIdx.x == 0) {
    *gave_up() = 0;
    for (int w = 0; w < TREE_WARPS; ++w)
      for (int i = 0; i < STAGES; ++i) mbar_init(smem_u32(&sm.full[w][i]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  int seq = 0;
  if (t.split == 0) {
    const int b = blockIdx.z;
    const KeyRange kr = key_range(t.c, b);
    if (!kr.rq.ok && threadIdx.x == 0) cache_report(t.c, CACHE_BAD_OFFSETS);
    const int row_tiles = tree_row_tiles(t, kr.rq.tokens), tiles = tree_key_tiles(t, kr.keys);
    for (int rt = blockIdx.x; rt < row_tiles; rt += gridDim.x) tree_mma_piece<DH, CAP>(t, map, sm, TreePiece{b, (int)blockIdx.y, rt, 0, tiles, tiles}, seq);
  } else {
    sm.plan.make(t);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the join's blocks may make their plan beside this
    if (blockIdx.x == 0)
      for (int b = threadIdx.x; b < t.c.batch; b += 32 * TREE_WARPS)
        if (!cache_request(t.c, b).ok) cache_report(t.c, CACHE_BAD_OFFSETS);
    const long long end = sm.plan.bound(blockIdx.x + 1);
    const long long start = sm.plan.bound(blockIdx.x);
    if (threadIdx.x == 0) t.join[blockIdx.x].rows = 0;
    for (long long pos = start; pos < end;) {
      const bool first = pos == start;
      long long unit_end;
      const TreePiece pc = sm.plan.piece(t, pos, end, &pos, &unit_end);
      if (first && threadIdx.x == 0) sm.plan.note_join(t, blockIdx.x, pc, unit_end);
      if (pc.begin < pc.end) tree_mma_piece<DH, CAP>(t, map, sm, pc, seq);
    }
  }
  if (*gave_up()) __nanosleep(1000000);                  // copies may still be on their way into this block's memory
}

// The parts of a unit that blocks x - 1, x, ... left, joined in the order of the keys: a block takes four rows at a time, one a warp or, of
// many parts, one after the other with every fourth part a warp
constexpr int JOIN_WARPS = 4;
template <int DH>
__global__ void __launch_bounds__(32 * JOIN_WARPS) tree_join_kernel(const TreeView t) {
  __shared__ float acc_of[JOIN_WARPS][DH];
  __shared__ float sum_of[JOIN_WARPS];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int x = blockIdx.x + 1, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const TreeJoin j = t.join[x];
  constexpr int PER = DH / 32;
  const int parts = j.to - x + 1;
  const bool alone = parts <= 2 * JOIN_WARPS;              // few parts: a warp takes a row for itself
  for (int row = alone ? blockIdx.y * JOIN_WARPS + warp : blockIdx.y; row < j.rows; row += gridDim.y * (alone ? JOIN_WARPS : 1)) {
      auto slot = [&](int k) { return ((long long)2 * (x - 1 + k) + (k == 0 ? 1 : 0)) * t.rows + row; };   // of part k
      float top = -INFINITY;
      for (int k = lane; k < parts; k += 32) top = fmaxf(top, t.part_ml[slot(k)].x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float base = top == -INFINITY ? 0.f : top;
      float sum = 0.f, acc[PER];
#pragma unroll
      for (int d = 0; d < PER; ++d) acc[d] = 0.f;
#pragma unroll 4
      for (int k = alone ? 0 : warp; k < parts; k += alone ? 1 : JOIN_WARPS) {
        const float2 ml = t.part_ml[slot(k)];
        const float* o = t.part_o + slot(k) * DH + lane * PER;
        const float f = tree_ex2(ml.x - base);
        sum += ml.y == 0.f ? 0.f : ml.y * f;
#pragma unroll
        for (int d = 0; d < PER; ++d) { const float v = o[d]; acc[d] += ml.y == 0.f ? 0.f : v * f; }   // a part that saw no key may hold anything
      }
      if (!alone) {
        __syncthreads();
        if (lane == 0) sum_of[warp] = sum;
#pragma unroll
        for (int d = 0; d < PER; ++d) acc_of[warp][lane * PER + d] = acc[d];
        __syncthreads();
        sum = 0.f;
#pragma unroll
        for (int d = 0; d < PER; ++d) acc[d] = 0.f;
#pragma unroll
        for (int w = 0; w < JOIN_WARPS; ++w) {
          sum += sum_of[w];
#pragma unroll
          for (int d = 0; d < PER; ++d) acc[d] += acc_of[w][lane * PER + d];
        }
        if (warp != 0) continue;
      }
      const int r = j.row0 + row, tk = r / t.group, head = j.h * t.group + r % t.group;
      uint16_t* const out = t.a.out + ((long long)(j.token0 + tk) * t.a.num_q_heads + head) * DH + lane * PER;
      uint16_t y[PER];
#pragma unroll
      for (int d = 0; d < PER; ++d) { const bf16 v = f2bf(sum == 0.f ? 0.f : acc[d] / sum); y[d] = *reinterpret_cast<const uint16_t*>(&v); }
      if (PER == 4) *reinterpret_cast<uint2*>(out) = make_uint2(y[0] | (uint32_t)y[1 % PER] << 16, y[2 % PER] | (uint32_t)y[3 % PER] << 16);
      else if (PER == 2) *reinterpret_cast<uint32_t*>(out) = y[0] | (uint32_t)y[1 % PER] << 16;
      else out[0] = y[0];
    }
}

template <int DH, int CAP>
phx_status tree_mma_launch(const TreeView& t, cudaStream_t stream, std::string& err) {
  constexpr int smem = (int)sizeof(TreeSmem<DH>) + 1024;
  static SmemLimit limit;
  PHX_CUDA_TRY(limit.raise(tree_mma_kernel<DH, CAP>, smem), err);
  CUtensorMap map;
  const phx_status st = tree_pool_map(&map, t, KEYS, err);
  if (st != PHX_OK) return st;
  const long long rows = (long long)t.a.max_tokens * t.group;
  const unsigned tiles = (unsigned)((rows + ROWS - 1) / ROWS < 65535 ? (rows + ROWS - 1) / ROWS : 65535);
  const dim3 grid = t.split ? dim3(t.split) : dim3(tiles, t.c.num_kv_heads, t.c.batch);
  tree_mma_kernel<DH, CAP><<<grid, 32 * TREE_WARPS, smem, stream>>>(t, map);
  PHX_CUDA_TRY(cudaGetLastError(), err);
  dispatch_note(DK_TREE_MMA);
  return PHX_OK;
}
template <int DH>
phx_status tree_mma_launch(const TreeView& t, cudaStream_t stream, std::string& err) {
  // Up to 1000 the exponential form's error, 1e-7 of the cap, is far below the bf16 rounding of the probabilities, and it is the faster one here: 76.6 us against 82.1 for 96
  // single tokens over up to 4096 keys, 103 against 105 (113 with logits around the cap) for prompts of 512 with heads of 32.
  if (t.a.cap_method == 2 && t.a.cap > 1000.0f) return tree_mma_launch<DH, WIDE_CAP>(t, stream, err);
  return t.a.cap_method == 0 ? tree_mma_launch<DH, 0>(t, stream, err) : t.a.cap_method == 1 ? tree_mma_launch<DH, 1>(t, stream, err) : tree_mma_launch<DH, 2>(t, stream, err);
}

long long part_bytes(int split, int rows, int dh) { return 2ll * split * rows * (dh * 4 + 8) + split * (long long)sizeof(TreeJoin); }

}  // namespace

// The pool as rows of key_size; a box is 64 (32) columns of `box_rows` rows, swizzled; rows behind the pool read as zeros
phx_status tree_pool_map(CUtensorMap* map, const TreeView& t, int box_rows, std::string& err) {
  EncodeTiledFn fn = get_encode_fn(err);
  if (!fn) return PHX_E_CUDA;
  const int dh = t.c.key_size;
  cuuint64_t dims[2] = {(cuuint64_t)dh, (cuuint64_t)(2 * t.c.num_pages * t.c.num_kv_heads * t.c.page_size)};
  cuuint64_t strides[1] = {(cuuint64_t)dh * 2};
  cuuint32_t box[2] = {(cuuint32_t)(dh < 64 ? dh : 64), (cuuint32_t)box_rows}, estr[2] = {1, 1};
  const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, t.c.pages, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        dh < 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) { err = "cuTensorMapEncodeTiled failed with code " + std::to_string((int)r); return PHX_E_CUDA; }
  return PHX_OK;
}

}  // namespace phx

using namespace phx;

extern "C" phx_status phx_tree_workspace_bytes(int32_t device, int64_t* bytes_out) {
  if (!bytes_out) { set_global_error("phx_tree_workspace_bytes: null argument"); return PHX_E_ARG; }
  DeviceScope scope(device);
  if (!scope.ok()) { set_global_error("phx_tree_workspace_bytes: cudaSetDevice failed"); return PHX_E_CUDA; }
  *bytes_out = part_bytes(tree_tc_blocks_per_sm() * device_sms(), 128, 128);   // the largest that a call may take
  return PHX_OK;
}

extern "C" phx_status phx_tree_attention_device(int32_t device, const phx_cache_batch* cache, const phx_tree_args* args, void* stream) {
  auto bad = [](const char* m) { set_global_error(std::string("phx_tree_attention_device: ") + m); return PHX_E_ARG; };
  const char* what = cache_check(cache);
  if (*what) return bad(what);
  if (!args) return bad("null argument");
  TreeView t;
  t.c = *cache; t.a = *args;
  if (t.a.num_q_heads < 1 || t.a.num_q_heads > 4096 || t.a.num_q_heads % t.c.num_kv_heads != 0) return bad("num_q_heads must be a multiple of num_kv_heads, at most 4096");
  if (t.a.cap_method < 0 || t.a.cap_method > 2) return bad("cap_method must be 0, 1 or 2");
  if (!isfinite(t.a.sm_scale) || !isfinite(t.a.cap)) return bad("sm_scale and cap must be finite");
  if (t.a.cap_method != 0 && !(t.a.cap > 0.f)) t.a.cap_method = 0;
  if (t.c.batch > 65535) return bad("at most 65535 requests");
  if (t.a.q_stride < (long long)t.a.num_q_heads * t.c.key_size || t.a.q_stride % 8 != 0) return bad("q_stride must be a multiple of 8 and cover a token's heads");
  if (t.a.max_tokens < 0 || t.a.max_keys < 0) return bad("negative size");
  if (t.c.batch == 0 || t.c.num_tokens == 0) return PHX_OK;
  if (t.a.max_tokens < 1) t.a.max_tokens = 1;
  if (t.a.max_tokens > t.c.num_tokens) t.a.max_tokens = t.c.num_tokens;
  if (!t.a.q || !t.a.out || !aligned16(t.a.q) || !aligned16(t.a.out)) return bad("q and out must be 16-byte aligned buffers");
  if ((reinterpret_cast<uintptr_t>(t.a.spans) & 7) != 0) return bad("spans must be 8-byte aligned");
  if (!t.a.workspace || !aligned16(t.a.workspace)) return bad("workspace must be a 16-byte aligned buffer");
  t.csc = t.a.sm_scale * TREE_LOG2E;
  t.group = t.a.num_q_heads / t.c.num_kv_heads;
  DeviceScope scope(device);
  if (!scope.ok()) { set_global_error("phx_tree_attention_device: cudaSetDevice failed"); return PHX_E_CUDA; }
  cudaStream_t st = (cudaStream_t)stream;
  std::string err;

  // More than 16 rows a key head are the tensor cores' (tree_attention_sm100.cu); the mma.sync kernel would read the cache again for every 16.
  const bool tc = tree_tc_supported(t) && (long long)t.a.max_tokens * t.group > ROWS;
  t.rows = ROWS; t.keys = KEYS * TREE_WARPS; t.setup = 2;
  if (tc) tree_tc_shape(t);
  const int per_sm = tc ? tree_tc_blocks_per_sm() : t.c.key_size == 128 ? mma_blocks<128>() : mma_blocks<64>();
  // Blocks share the tiles of all units where there are few units for them and long ones among them.  Measured on the tensor cores (us, shared / whole): 2 to 3
  // units a block, heads of 128, with 0.4 of the last round's blocks empty and 16, 64, 128 tiles a unit 108 / 87, 285 / 273, 523 / 523; with 0.84 empty 97 / 82, 245 / 253,
  // 443 / 482; with none 104 / 94, 307 / 299, 575 / 564.  Heads of 64, 0.4 empty: 81 / 64, 193 / 196, 356 / 377;
  // 0.84 empty and 32, 64, 128 tiles: 102 / 98, 166 / 177, 299 / 340.  Whole ones cost the empty blocks; shared ones the parts and their join, as wide as a head:
  // about 48 tiles for 128, 24 for 64.  Up to two a block they are shared all the same: lengths are seldom equal.
  const long long units = (long long)t.c.batch * t.c.num_kv_heads * (((long long)t.a.max_tokens * t.group + t.rows - 1) / t.rows);
  const long long tiles = (t.a.max_keys + t.keys - 1) / t.keys;
  const long long blocks = per_sm * device_sms(), fed = units * (tiles + t.setup) / (tc ? 8 : 4);   // no block for fewer places: parts and joins take longer than that many
  const long long idle = (units + blocks - 1) / blocks * blocks - units;                  // blocks without a unit in the last round of whole ones
  const bool few = tc ? tiles >= 8 && (units < 2 * blocks || idle * tiles > 3 * t.c.key_size / 8 * blocks) : tiles >= 4 && units < 8 * blocks;
  t.split = few && t.c.batch <= TREE_MAX_SPLIT_BATCH ? (int)(fed < blocks ? fed : blocks) : 0;
  if (t.split < 2) t.split = 0;                                                            // one block takes whole units: there is no bound between blocks, nothing to join
  t.turns = tc && !t.split && units > blocks && t.c.batch <= TREE_MAX_SPLIT_BATCH ? (int)blocks : 0;
  if (part_bytes(t.split, t.rows, t.c.key_size) > t.a.workspace_bytes) return bad("workspace is smaller than phx_tree_workspace_bytes");
  t.part_o = static_cast<float*>(t.a.workspace);
  t.part_ml = reinterpret_cast<float2*>(t.part_o + 2ll * t.split * t.rows * t.c.key_size);
  t.join = reinterpret_cast<TreeJoin*>(t.part_ml + 2ll * t.split * t.rows);
  if (t.c.num_pages == 0) return bad("an empty pool has no keys to attend to");
  phx_status s = tc ? tree_tc_launch(t, st, err) : t.c.key_size == 32 ? tree_mma_launch<32>(t, st, err) : t.c.key_size == 64 ? tree_mma_launch<64>(t, st, err) : tree_mma_launch<128>(t, st, err);
  if (s == PHX_OK && t.split) {
    const long long rows = (long long)t.a.max_tokens * t.group;
    const unsigned most = (unsigned)(rows < t.rows ? rows : t.rows);
    const bool many = t.split > JOIN_WARPS * units;                // parts of a unit: a block for each row, else for four
    const dim3 grid(t.split - 1, many ? most : (most + JOIN_WARPS - 1) / JOIN_WARPS), block(32 * JOIN_WARPS);
    const cudaError_t e = t.c.key_size == 32 ? launch_programmatic(tree_join_kernel<32>, grid, block, 0, st, t)
                          : t.c.key_size == 64 ? launch_programmatic(tree_join_kernel<64>, grid, block, 0, st, t)
                                               : launch_programmatic(tree_join_kernel<128>, grid, block, 0, st, t);
    if (e != cudaSuccess) { err = cudaGetErrorString(e); s = PHX_E_CUDA; }
  }
  if (s != PHX_OK) {
    (void)cudaGetLastError();
    set_global_error("phx_tree_attention_device: " + err);
  }
  return s;
}

// Depth-first places of a forest given by parents, without recursion: tokens below each token are counted from the leaves up
// (a topological order from the number of children left), then every parent hands its children their places from the roots down.
extern "C" phx_status phx_tree_spans(const int32_t* parents, int32_t n, int32_t* spans_out) {
  auto bad = [](const char* m) { set_global_error(std::string("phx_tree_spans: ") + m); return PHX_E_ARG; };
  if (n < 0 || (n > 0 && (!parents || !spans_out))) return bad("null argument or negative size");
  try {
    std::vector<int32_t> open((size_t)n, 0), below((size_t)n, 1), order;
    order.reserve((size_t)n);
    for (int32_t i = 0; i < n; ++i) {
      const int32_t p = parents[i];
      if (p < -2 || p >= n || p == i || (p >= 0 && parents[p] == -2)) return bad("a parent must be -1, -2 (padding) or another token that is no padding");
      if (p >= 0) ++open[p];
    }
    for (int32_t i = 0; i < n; ++i) if (open[i] == 0) order.push_back(i);
    for (size_t at = 0; at < order.size(); ++at) {
      const int32_t i = order[at], p = parents[i];
      if (p >= 0) { below[p] += below[i]; if (--open[p] == 0) order.push_back(p); }
    }
    if ((int32_t)order.size() != n) return bad("the parents form a cycle");
    std::vector<int32_t> next((size_t)n, 0);
    int32_t top = 0;
    for (int32_t i = 0; i < n; ++i)   // roots take their places in the order of the tokens
      if (parents[i] == -1) { spans_out[2 * i] = top; top += below[i]; spans_out[2 * i + 1] = top; next[i] = spans_out[2 * i] + 1; }
      else if (parents[i] == -2) spans_out[2 * i] = spans_out[2 * i + 1] = -1;
    for (size_t at = order.size(); at-- > 0;) {   // parents come behind their children in `order`
      const int32_t i = order[at], p = parents[i];
      if (p < 0) continue;
      spans_out[2 * i] = next[p];
      next[p] += below[i];
      spans_out[2 * i + 1] = next[p];
      next[i] = spans_out[2 * i] + 1;
    }
  } catch (const std::exception& e) {
    set_global_error(std::string("phx_tree_spans: ") + e.what());
    return PHX_E_CAPACITY;
  }
  return PHX_OK;
}
