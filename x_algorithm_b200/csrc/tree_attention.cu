// Attention of a request's new tokens over its paged cache, their own keys included (phx_tree_attention_device):
//
//   o_i = sum_j p_ij v_j,   p_ij = softmax over the keys j that i sees of cap(q_i . k_j * scale)
//
// i sees every key cached before, and of the new tokens' keys those with pre[j] <= pre[i] < end[j].  The g query heads that share
// a key head are rows of one product: row r of a request and key head is token r / g, head r % g of the group, so K and V are read
// once for all of them.
//
// The mma.sync kernel: a CTA's four warps share 16 such rows and take 32 keys each in turn, every warp with its own ring of key and value
// tiles (cp.async, 16 bytes a piece, no barrier between the warps), running maximum, sum and output; they are joined once at the end.  Masked logits
// become -inf before the maximum; a value row that some of the tile's rows do not see must not reach them as 0 * NaN either, so tiles that are
// not seen whole are searched for infinities and NaN, which are then added to the rows that do see them, one by one.
#include <string>
#include <vector>

#include "cache_batch.cuh"

namespace phx {
namespace {

constexpr int TREE_WARPS = 4;
constexpr int ROWS = 16;         // query rows of a tile
constexpr int KEYS = 32;         // keys of a warp's tile
constexpr int STAGES = 3;
constexpr float LOG2E = 1.4426950408889634f;

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
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool there) {   // not there: 16 zero bytes
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ bool odd_value(uint16_t v) { return (v & 0x7F80u) == 0x7F80u; }   // infinity or NaN
__device__ __forceinline__ bool odd_pair(uint32_t v) { return (v & 0x7F80u) == 0x7F80u || (v & 0x7F800000u) == 0x7F800000u; }

// byte of 16-byte piece `piece` of row `row` in a tile: rows of DH * 2 bytes, pieces exchanged so that the eight rows of an ldmatrix
// block fall on different banks
template <int DH>
__device__ __forceinline__ uint32_t tile_at(int row, int piece) {
  constexpr int PIECES = DH / 8;
  const int sw = PIECES >= 8 ? (row & 7) : ((row >> 1) & 3);
  return (uint32_t)(row * DH * 2 + ((piece ^ sw) << 4));
}

struct TreeView {
  phx_cache_batch c;
  phx_tree_args a;
  float csc;           // scale into the log2 domain (no cap)
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

template <int DH>
struct TreeSmem {
  uint8_t kv[TREE_WARPS][STAGES][2][KEYS * DH * 2];
  int tile[TREE_WARPS][STAGES];
  int there[TREE_WARPS][STAGES];   // bit i: keys 16 i .. 16 i + 15 of the tile sit in a page of the pool
  float m[TREE_WARPS][ROWS], l[TREE_WARPS][ROWS];
};

template <int DH, int CAP>
__global__ void __launch_bounds__(32 * TREE_WARPS) tree_mma_kernel(const TreeView t) {
  extern __shared__ __align__(128) uint8_t smem_bytes[];
  TreeSmem<DH>& sm = *reinterpret_cast<TreeSmem<DH>*>(smem_bytes);
  constexpr int PIECES = DH / 8, KSTEPS = DH / 16, NT = DH / 8;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.y, b = blockIdx.z;
  const KeyRange kr = key_range(t.c, b);
  const CacheRequest& rq = kr.rq;
  const int group = t.a.num_q_heads / t.c.num_kv_heads;
  const long long rows = (long long)rq.tokens * group;
  const int n_tiles = (kr.keys + KEYS - 1) / KEYS;
  if (threadIdx.x == 0 && (!rq.ok || kr.keys < (long long)rq.cached + rq.tokens)) cache_report(t.c, rq.ok ? CACHE_BAD_PAGE : CACHE_BAD_OFFSETS);
  const long long v_off = (long long)t.c.num_kv_heads * t.c.page_size * DH;   // from a key to its value
  const uint32_t kv_smem = (uint32_t)__cvta_generic_to_shared(sm.kv[warp]);

  for (long long r0 = (long long)blockIdx.x * ROWS; r0 < rows; r0 += (long long)gridDim.x * ROWS) {
    // rows lane / 4 and lane / 4 + 8 of the tile: token, its place in the walk, A fragments of the query
    int tok[2], pre[2];
    const uint16_t* qrow[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const long long r = min(r0 + lane / 4 + 8 * i, rows - 1);
      tok[i] = (int)(r / group);
      const int head = h * group + (int)(r - (long long)tok[i] * group);
      pre[i] = span_of(t, rq, tok[i]).x;
      qrow[i] = t.a.q + (long long)(rq.row0 + tok[i]) * t.a.q_stride + head * DH;
    }
    uint32_t q[KSTEPS][4];
#pragma unroll
    for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        q[k][i] = *reinterpret_cast<const uint32_t*>(qrow[i & 1] + k * 16 + (i >> 1) * 8 + (lane & 3) * 2);
    // the places that the tile's rows take in the walk: a tile of new keys that none of them sees is not loaded
    int lo = min(pre[0] < 0 ? 0x7fffffff : pre[0], pre[1] < 0 ? 0x7fffffff : pre[1]), hi = max(pre[0], pre[1]);
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) { lo = min(lo, __shfl_xor_sync(0xffffffffu, lo, o)); hi = max(hi, __shfl_xor_sync(0xffffffffu, hi, o)); }

    float acc[NT][4];
#pragma unroll
    for (int i = 0; i < NT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

    int next = warp;                                   // the next tile of this warp that may be needed
    auto load = [&](int stage) {                       // its copy into `stage`, or a note that there is none
      int tile = -1;
      for (; next < n_tiles; next += TREE_WARPS) {
        const int j = next * KEYS + lane - rq.cached;  // this lane's key among the new ones
        bool seen = next * KEYS + lane < kr.keys;
        if (seen && j >= 0) { const int2 s = span_of(t, rq, j); seen = s.x <= hi && s.y > lo; }
        if (__any_sync(0xffffffffu, seen && hi >= 0)) { tile = next; next += TREE_WARPS; break; }
      }
      if (tile >= 0) {
        int there = 0;
        long long at[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {                  // 16 keys never cross a page
          const int key = tile * KEYS + 16 * i, col = key / t.c.page_size;
          const int page = key < kr.keys ? kr.table[col] : 0;
          const bool ok = key < kr.keys && page >= 0 && page < t.c.num_pages;
          if (key < kr.keys && !ok && lane == 0) cache_report(t.c, CACHE_BAD_PAGE);
          there |= ok ? 1 << i : 0;
          at[i] = ok ? cache_row0(t.c, page, 0, h) + (long long)(key - col * t.c.page_size) * DH : 0;
        }
        const uint32_t dst = kv_smem + stage * (2 * KEYS * DH * 2);
#pragma unroll
        for (int i = 0; i < KEYS * PIECES / 32; ++i) {
          const int row = (i * 32 + lane) / PIECES, piece = (i * 32 + lane) % PIECES;
          const bool ok = ((there >> (row >> 4)) & 1) && tile * KEYS + row < kr.keys;
          const uint16_t* src = t.c.pages + (ok ? at[row >> 4] + (row & 15) * DH + piece * 8 : 0);
          cp16(dst + tile_at<DH>(row, piece), src, ok);
          cp16(dst + KEYS * DH * 2 + tile_at<DH>(row, piece), src + (ok ? v_off : 0), ok);
        }
        if (lane == 0) sm.there[warp][stage] = there;
      }
      if (lane == 0) sm.tile[warp][stage] = tile;
      asm volatile("cp.async.commit_group;" ::: "memory");
    };

#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) load(s);
    for (int it = 0;; ++it) {
      const int stage = it % STAGES;
      load((it + STAGES - 1) % STAGES);
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
      __syncwarp();
      const int tile = sm.tile[warp][stage];
      if (tile < 0) break;
      const int there = sm.there[warp][stage];
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
      const bool whole = key0 + KEYS <= min(rq.cached, kr.keys) && there == 3;
      uint32_t seen[2] = {0xffu, 0xffu};               // bit 2 n + c: key 8 n + (lane & 3) * 2 + c, for either row
#pragma unroll
      for (int n = 0; n < KEYS / 8; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float v = s[n][c];
          if (CAP == 0) v *= t.csc;
          else if (CAP == 1) { v *= t.a.sm_scale; v = v / (1.0f + fabsf(v) / t.a.cap) * LOG2E; }
          else { v *= t.a.sm_scale; v = t.a.cap * tanhf(v / t.a.cap) * LOG2E; }
          s[n][c] = v;
        }
      if (!whole) {
        seen[0] = seen[1] = 0;
#pragma unroll
        for (int n = 0; n < KEYS / 8; ++n)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int in = n * 8 + (lane & 3) * 2 + c, key = key0 + in;
            const bool ok = key < kr.keys && ((there >> (in >> 4)) & 1);
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
        const float mn = fmaxf(m[i], mx), base = mn == -INFINITY ? 0.f : mn, alpha = ex2(m[i] - base);
        m[i] = mn;
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < KEYS / 8; ++n) {
          const float e0 = ex2(s[n][2 * i] - base), e1 = ex2(s[n][2 * i + 1] - base);
          sum += e0 + e1;
          p[n >> 1][(n & 1) * 2 + i] = pack_bf2(e0, e1);   // rounded to bf16 for the product; the sum keeps fp32
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
              if (odd_value((uint16_t)v[k])) v[k] &= 0xffff0000u;
              if (odd_value((uint16_t)(v[k] >> 16))) v[k] &= 0xffffu;
            }
            asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
          }
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
    asm volatile("cp.async.wait_group 0;" ::: "memory");

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
        const float f = ex2(sm.m[w][row] - base);
        if (sm.l[w][row] == 0.f) continue;                         // a part that saw no key
        sum += sm.l[w][row] * f;
        const float* src = part + (w * ROWS + row) * DH + piece * 8;
#pragma unroll
        for (int k = 0; k < 8; ++k) o[k] += src[k] * f;
      }
      const long long r = r0 + row;
      const int tk = (int)(r / group), head = h * group + (int)(r % group);
      const bool none = sum == 0.f || span_of(t, rq, tk).x < 0;    // no key seen, or a padding token
      const float inv = none ? 0.f : 1.0f / sum;
#pragma unroll
      for (int k = 0; k < 8; ++k) o[k] = none ? 0.f : o[k] * inv;
      const uint4 v = make_uint4(pack_bf2(o[0], o[1]), pack_bf2(o[2], o[3]), pack_bf2(o[4], o[5]), pack_bf2(o[6], o[7]));
      *reinterpret_cast<uint4*>(t.a.out + ((long long)(rq.row0 + tk) * t.a.num_q_heads + head) * DH + piece * 8) = v;
    }
    __syncthreads();
  }
}

template <int DH, int CAP>
cudaError_t tree_mma_launch(const TreeView& t, cudaStream_t stream) {
  static SmemLimit limit;
  cudaError_t e = limit.raise(tree_mma_kernel<DH, CAP>, (int)sizeof(TreeSmem<DH>));
  if (e != cudaSuccess) return e;
  const long long rows = (long long)t.a.max_tokens * (t.a.num_q_heads / t.c.num_kv_heads);
  const unsigned tiles = (unsigned)((rows + ROWS - 1) / ROWS < 65535 ? (rows + ROWS - 1) / ROWS : 65535);
  tree_mma_kernel<DH, CAP><<<dim3(tiles, t.c.num_kv_heads, t.c.batch), 32 * TREE_WARPS, sizeof(TreeSmem<DH>), stream>>>(t);
  return cudaGetLastError();
}
template <int DH>
cudaError_t tree_mma_launch(const TreeView& t, cudaStream_t stream) {
  return t.a.cap_method == 0 ? tree_mma_launch<DH, 0>(t, stream) : t.a.cap_method == 1 ? tree_mma_launch<DH, 1>(t, stream) : tree_mma_launch<DH, 2>(t, stream);
}

}  // namespace
}  // namespace phx

using namespace phx;

extern "C" phx_status phx_tree_workspace_bytes(int32_t device, int64_t* bytes_out) {
  if (!bytes_out) { set_global_error("phx_tree_workspace_bytes: null argument"); return PHX_E_ARG; }
  (void)device;
  *bytes_out = 0;
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
  if (!(t.a.sm_scale == t.a.sm_scale) || !(t.a.cap == t.a.cap)) return bad("sm_scale and cap must be numbers");
  if (t.a.cap_method != 0 && !(t.a.cap > 0.f)) t.a.cap_method = 0;
  if (t.c.batch > 65535) return bad("at most 65535 requests");
  if (t.a.q_stride < (long long)t.a.num_q_heads * t.c.key_size || t.a.q_stride % 8 != 0) return bad("q_stride must be a multiple of 8 and cover a token's heads");
  if (t.a.max_tokens < 0 || t.a.max_keys < 0) return bad("negative size");
  if (t.c.batch == 0 || t.c.num_tokens == 0) return PHX_OK;
  if (t.a.max_tokens < 1) t.a.max_tokens = 1;
  if (!t.a.q || !t.a.out || !aligned16(t.a.q) || !aligned16(t.a.out)) return bad("q and out must be 16-byte aligned buffers");
  if ((reinterpret_cast<uintptr_t>(t.a.spans) & 7) != 0) return bad("spans must be 8-byte aligned");
  t.csc = t.a.sm_scale * LOG2E;
  DeviceScope scope(device);
  if (!scope.ok()) { set_global_error("phx_tree_attention_device: cudaSetDevice failed"); return PHX_E_CUDA; }
  cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = t.c.key_size == 32 ? tree_mma_launch<32>(t, st) : t.c.key_size == 64 ? tree_mma_launch<64>(t, st) : tree_mma_launch<128>(t, st);
  if (e != cudaSuccess) { set_global_error(std::string("phx_tree_attention_device: ") + cudaGetErrorString(e)); return PHX_E_CUDA; }
  dispatch_note(DK_TREE_MMA);
  return PHX_OK;
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
