// Log probabilities of given ids, entropy and best alternatives from a row of logits (phx_token_logprobs_device):
//
//   c = cap tanh(x / cap),  d = c - max c,  t = d / temperature,  Z = sum e^t
//   log p = t - ln Z,   entropy = ln Z - sum e^t t / Z
//
// The maximum is taken off before anything else, so that neither rows of a type's lowest value nor large logits overflow or cancel.
//
// One pass over the logits, bound by memory.  A row belongs to a warp, to a block, or to a cluster of blocks that each take a
// stretch of it.  A thread fetches its own 16-byte words, cp.async into a ring of its own in shared memory (no barriers), takes a few
// of them at a time, and keeps a reference, the sum of e^t and the sum of e^t t against it.  The reference is the running maximum of the warp: the best id's
// own exponential is 1 at the end, and its log p near 0 is good to 1e-7 (a reference that may be 11 below it cost 1e-6).  It moves a few times a row; a lane's
// own maximum moved in some lane of a warp at almost every batch, a third of the instructions.
//
// The best ids are found by words first: a word's key is its largest logit's order-preserving image, then its place, first come first.
// The top_k-th largest key of any set of words bounds what the row's best ids can be in - a word below it holds nothing that is not
// beaten by a logit in each of top_k other words - so after the first batch the threads' best words give a bound, and from then on the words at
// or above it, few, are noted in shared memory.  After 2, 4, 8, ... batches the bound is taken anew from the notes, if they
// fill a quarter of their room, and the rest is dropped.  At the end the notes' words are
// read again, their (logit, id) keys bounded in the same way, and the survivors ranked by counting.  Rows whose order defeats the
// bounds (sorted ones: more words than the notes hold) take the exact bound from a radix select over the keys, a byte a pass.  Keys are
// distinct, so ties need no care and the result does not depend on the order of the atomics.  More ids than lanes give a bound for (over 24) of
// a row that a warp has for itself are found exactly: the row's images in registers, their top_k-th largest by halving.
//
// Measured: 2048 rows of 100003 bf16 logits 83 us = 4.9 TB/s without best ids, 117 with eight, 150 and 180 capped; 1024 rows of 100004 fp32 72 us = 5.6 TB/s and 85;
// one row of 131072 fp32, best 20, 11.9 us on eight blocks.  The selection behind a row's last word is what the eight cost.  A cap that logits reach costs more: beyond 3/4 of it a
// thread takes its batch one by one, 630 us for the 2048 rows with logits of 4 times a standard normal under a cap of 10.
#include <math.h>
#include <string.h>

#include <string>

#include "cache_batch.cuh"

namespace phx {
namespace {

constexpr int WARP_ROWS = 4;        // rows of a block whose warps take one each
constexpr int WARP_ROW = 1024;      // the longest of them
constexpr float LOG2E = 1.4426950408889634f;
constexpr float FLOOR = -1e38f, DEEP = -1e37f;
typedef unsigned long long u64;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {   // NaN if either is
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float warp_max_nan(float x) {       // of a warp's lanes
  float y;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
// order-preserving: larger logit, larger image; the two zeros are equal, NaN is largest
__device__ __forceinline__ uint32_t image(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ u64 key_of(float x, int id) { return ((u64)image(x) << 32) | (uint32_t)~id; }
__device__ __forceinline__ float value_of(u64 key) {           // the logit of a key
  const uint32_t u = (uint32_t)(key >> 32);
  return u == 0xFFFFFFFFu ? NAN : __uint_as_float(u & 0x80000000u ? u & 0x7FFFFFFFu : ~u);
}

template <typename T> struct Words;   // elements of a 16-byte word
template <> struct Words<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& v, float* x) {
    x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
  }
  static __device__ __forceinline__ float at(const float* row, long long i) { return row[i]; }
};
template <> struct Words<bf16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
  }
  static __device__ __forceinline__ float at(const bf16* row, long long i) { return bf2f(row[i]); }
};

// m the reference, d = c - m: z = sum of e^t, s = sum of e^t d
struct Stat { float m, z, s; };
__device__ __forceinline__ Stat join(const Stat& a, const Stat& b, float scale) {
  Stat r;
  r.m = max_nan(a.m, b.m);
  const float base = r.m == -INFINITY ? 0.f : r.m;
  const float da = a.m - base, db = b.m - base, fa = ex2(da * scale), fb = ex2(db * scale);
  r.z = a.z * fa + b.z * fb;
  r.s = (fa == 0.f ? 0.f : fa * (a.s + a.z * da)) + (fb == 0.f ? 0.f : fb * (b.s + b.z * db));   // e^t d is 0 where e^t is
  return r;
}
// cap tanh(x / cap); -inf stays -inf.  Small logits, |x| <= 3/4 cap, by an odd polynomial in x / cap (least maximum error 1e-8 of the cap, found by reweighted
// least squares on Chebyshev nodes): four logits take it in the time of one tanhf.  The sums and the answers use the same function: with a faster one for the sums alone, off
// by 1e-7 of the cap, log probabilities near 0 were off by 1e-5 of themselves.
struct Cap {
  float cap, most, c[6];
  // (below 1e-3 the powers of 1 / cap leave fp32: no logit counts as small there)
  __device__ __forceinline__ explicit Cap(float limit) : cap(limit), most(limit >= 1e-3f ? 0.75f * limit : -1.0f) {
    const float z = 1.0f / limit, z2 = z * z;
    c[0] = 0.999999832f; c[1] = -0.333324709f * z2; c[2] = 0.133205796f * z2 * z2; c[3] = -0.0531492588f * z2 * z2 * z2;
    c[4] = 0.0192372317f * z2 * z2 * z2 * z2; c[5] = -0.0044934523f * z2 * z2 * z2 * z2 * z2;
  }
  __device__ __forceinline__ float small(float x) const {
    const float s = x * x;
    return x * fmaf(fmaf(fmaf(fmaf(fmaf(c[5], s, c[4]), s, c[3]), s, c[2]), s, c[1]), s, c[0]);
  }
  __device__ __forceinline__ float of(float x) const {
    if (fabsf(x) <= most) return small(x);
    return x == -INFINITY ? x : cap * tanhf(x / cap);
  }
};

// the threads that share a stretch of a row
template <int NT> struct Team {
  static __device__ __forceinline__ int tid() { return NT == 32 ? threadIdx.x & 31 : threadIdx.x; }
  static __device__ __forceinline__ void sync() { if (NT == 32) __syncwarp(); else __syncthreads(); }
};

template <int NT, int KEEP, int WORDS> struct TeamMemory {
  uint4 word[WORDS][NT];     // the rings; at the end, keys of single logits
  u64 keep[KEEP];                   // keys of words
  u64 group[NT], bounds[32];
  Stat part[NT / 32];
  int hist[256];
  int count;
  // what a block of a cluster hands to the first
  Stat stat;
  u64 best[PHX_LOGPROBS_MAX_TOP];
};

// A lower bound of the k-th largest of all keys that the team has, from each thread's largest (0: it has none).  k of 24 or fewer: the
// k-th largest of the maxima of 32 groups of threads; about 32 ln(32 / (32 - k)) keys of a random order lie at or above it.  More: with r the rank
// that three quarters of the warps need for k keys, the r-th largest of each warp's threads, and of these the one that leaves k.  Ranks by counting
// over 32 keys: over all the threads' it took longer than the logits.  Every call is followed by a barrier before the next.
template <int NT, typename M>
__device__ __forceinline__ u64 bound_of(u64 mine, int k, M& mem) {
  typedef Team<NT> G;
  constexpr int W = NT / 32;
  const int lane = threadIdx.x & 31, tid = G::tid();
  const bool few = W == 1 || k <= 24;
  if (few) {
#pragma unroll
    for (int o = 1; o < W; o <<= 1) { const u64 other = __shfl_xor_sync(0xffffffffu, mine, o); mine = other > mine ? other : mine; }
    if ((lane & (W - 1)) == 0) mem.group[tid / W] = mine;
    G::sync();
    if (tid >= 32) { G::sync(); return mem.bounds[0]; }
    mine = mem.group[lane];
  } else {
    mem.group[tid] = mine;
    __syncwarp();
  }
  const u64* const rivals = mem.group + (few ? 0 : tid & ~31);
  const int r = few ? k : (k + W * 3 / 4 - 1) / (W * 3 / 4);
  int above = 0;
#pragma unroll
  for (int j = 0; j < 32; ++j) above += rivals[j] > mine;
  const unsigned who = __ballot_sync(0xffffffffu, above == r - 1 && mine != 0);
  u64 bound = who == 0 ? 0 : __shfl_sync(0xffffffffu, mine, __ffs(who) - 1);
  if (few) {
    if (W > 1) {
      if (lane == 0) mem.bounds[0] = bound;
      G::sync();
    }
    return bound;
  }
  if (lane == 0) mem.bounds[tid >> 5] = bound;
  G::sync();
  const int q = (k + r - 1) / r;                 // warps that give k keys together
  bound = lane < W ? mem.bounds[lane] : 0;
  above = 0;
  for (int j = 0; j < W; ++j) above += mem.bounds[j] > bound || (mem.bounds[j] == bound && j < lane);
  const unsigned which = __ballot_sync(0xffffffffu, lane < W && above == q - 1);
  return __shfl_sync(0xffffffffu, bound, __ffs(which) - 1);
}

__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release;\n barrier.cluster.wait.acquire;" ::: "memory"); }
template <typename V>
__device__ __forceinline__ V* in_block(V* p, uint32_t rank) {   // the same place in another block of the cluster
  u64 out;
  asm volatile("mapa.u64 %0, %1, %2;" : "=l"(out) : "l"((u64)(uintptr_t)p), "r"(rank));
  return reinterpret_cast<V*>((uintptr_t)out);
}

// shape of a team: words it notes (all of a warp's row), words that a thread takes at a time, such batches in its ring, blocks that share an SM
template <int NT> struct Shape {
  static constexpr int KEEP = NT == 32 ? 320 : 1024, BATCH = NT == 256 ? 4 : 2, RING = NT == 32 ? 3 : 2, RESIDENT = NT == 1024 ? 1 : 4;
  typedef TeamMemory<NT, KEEP, RING * BATCH> Memory;
};

template <typename T, int NT, bool CAP>
__global__ void __launch_bounds__(NT == 32 ? 32 * WARP_ROWS : NT, Shape<NT>::RESIDENT) logprobs_kernel(const phx_logprobs_args a, int blocks) {
  constexpr int N = Words<T>::N, KEEP = Shape<NT>::KEEP, RING = Shape<NT>::RING, BATCH = Shape<NT>::BATCH;
  constexpr int SINGLE = RING * BATCH * NT * 2;             // keys of single logits that the rings' memory holds
  typedef Team<NT> G;
  typedef typename Shape<NT>::Memory Memory;
  extern __shared__ __align__(16) uint8_t smem_bytes[];
  Memory& mem = reinterpret_cast<Memory*>(smem_bytes)[NT == 32 ? threadIdx.x >> 5 : 0];
  const int r = NT == 32 ? blockIdx.x * WARP_ROWS + (threadIdx.x >> 5) : blockIdx.x / blocks;
  if (r >= a.rows) return;                                  // whole warps only
  const uint32_t rank = NT == 32 || blocks == 1 ? 0 : cluster_rank();
  const int tid = G::tid(), lane = threadIdx.x & 31, warp = tid >> 5;
  const T* const row = static_cast<const T*>(a.logits) + (long long)r * a.stride;
  const float scale = LOG2E / a.temperature;
  const bool flat = FLOOR * scale > -150.0f;                // a temperature (above 1e36) at which a distance of FLOOR would weigh something
  const Cap cap(CAP ? a.cap : 1.0f);

  // 16-byte words of the row, the first and last of them perhaps in part
  const int off = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  const T* const base = row - off;
  const int words = (int)(((long long)off + a.vocab + N - 1) / N), share = (words + blocks - 1) / blocks;
  const int w_begin = min((int)rank * share, words), w_end = min(w_begin + share, words);
  const int whole_begin = off > 0 ? 1 : 0, whole_end = (int)(((long long)off + a.vocab) / N);   // words that lie in the row with all their elements
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(&mem.word[0][tid]);
  // batch `it` of this thread - words w_begin + (it * BATCH + i) * NT + tid - on its way into the ring; what is not of the row is -inf
  auto fetch = [&](int it) {
    const int slot = (it % RING) * BATCH;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int w = w_begin + (it * BATCH + i) * NT + tid;
      const uint32_t dst = ring + (uint32_t)((slot + i) * NT) * 16u;
      if (w >= whole_begin && w < min(whole_end, w_end)) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(reinterpret_cast<const uint4*>(base) + w) : "memory");
      } else {
        const uint32_t none = N == 8 ? 0xFF80FF80u : 0xFF800000u;
        uint4* const slow = &mem.word[slot + i][tid];
        *slow = make_uint4(none, none, none, none);
        if (w < w_end)
#pragma unroll 1
          for (int k = 0; k < N; ++k)
            if (w * N - off + k >= 0 && w * N - off + k < a.vocab) reinterpret_cast<T*>(slow)[k] = row[w * N - off + k];
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };

  // the first given id of this thread and its logit, on their way under the row
  long long given_id = -1;
  float given_x = 0.f;
  if (a.given_out && rank == 0 && tid < a.num_given) {
    given_id = a.given[(long long)r * a.num_given + tid];
    if (given_id >= 0 && given_id < a.vocab) given_x = Words<T>::at(row, given_id);
  }

  Stat st = {-INFINITY, 0.f, 0.f};
  const bool want_top = a.top_k > 0 && (a.top_out || a.top_ids_out), exactly = NT == 32 && a.top_k > 24;
  u64 bound = ~0ull;              // of words
  float bound_x = INFINITY;       // its logit
  bool lost = false;              // more words than the notes hold
  if (tid == 0) mem.count = 0;
  G::sync();
  // a place behind what has been counted for each lane of a whole warp that wants one
  auto place_for = [&](bool want) {
    const unsigned who = __ballot_sync(0xffffffffu, want);
    int at = 0;
    if (lane == 0 && who != 0) at = atomicAdd(&mem.count, __popc(who));
    return __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1));
  };
  // keeps those of the keys `list` [n] that reach a bound taken from them, and the bound; between barriers
  auto tighten = [&](u64* list, int n) {
    u64 most = 0;
    for (int i = tid; i < n; i += NT) most = list[i] > most ? list[i] : most;
    u64 least = bound_of<NT>(most, a.top_k, mem);
    G::sync();
    if (tid == 0) mem.count = 0;
    G::sync();
    for (int i0 = 0; i0 < n; i0 += NT) {                         // in place: a key never moves up
      const u64 key = i0 + tid < n ? list[i0 + tid] : 0;
      G::sync();
      const bool stays = key != 0 && key >= least;
      const int at = place_for(stays);
      if (stays) list[at] = key;
      G::sync();
    }
    return least;
  };

  const int batches = (w_end - w_begin + BATCH * NT - 1) / (BATCH * NT);
#pragma unroll
  for (int i = 0; i < RING - 1; ++i) fetch(i);
  int again = 2;
#pragma unroll 1
  for (int it = 0; it < batches; ++it) {
    fetch(it + RING - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(RING - 1) : "memory");
    const int slot = (it % RING) * BATCH, w0 = w_begin + it * BATCH * NT + tid;
    uint4 cur[BATCH];
    float tops[BATCH], top = -INFINITY;     // of each word, of the batch; NaN if there is one
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(cur[i].x), "=r"(cur[i].y), "=r"(cur[i].z), "=r"(cur[i].w) : "r"(ring + (uint32_t)((slot + i) * NT) * 16u) : "memory");
      if (N == 8) {
        const uint32_t v[4] = {cur[i].x, cur[i].y, cur[i].z, cur[i].w};
        auto two = [&](int k) { return *reinterpret_cast<const __nv_bfloat162*>(&v[k]); };
        const __nv_bfloat162 m2 = __hmax2_nan(__hmax2_nan(two(0), two(1)), __hmax2_nan(two(2), two(3)));
        tops[i] = max_nan(__low2float(m2), __high2float(m2));
      } else {
        float x[N];
        Words<T>::unpack(cur[i], x);
        tops[i] = max_nan(max_nan(x[0], x[1]), max_nan(x[2], x[3]));
      }
      top = max_nan(top, tops[i]);
    }

    if (want_top && !exactly) {
      if (it == 0) {              // the first bound
        u64 best = 0;
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
          const u64 key = key_of(tops[i], w0 + i * NT);
          if (w0 + i * NT < w_end && key > best) best = key;
        }
        bound = bound_of<NT>(best, a.top_k, mem);
        bound_x = bound == 0 ? -INFINITY : value_of(bound);
      }
      if (!(top < bound_x)) {
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
          if (tops[i] < bound_x || w0 + i * NT >= w_end) continue;
          const u64 key = key_of(tops[i], w0 + i * NT);
          if (key >= bound) { const int at = atomicAdd(&mem.count, 1); if (at < KEEP) mem.keep[at] = key; }
        }
      }
      if (NT > 32 && it + 1 == again && it + 1 < batches) {          // a closer bound from what is there
        again *= 2;
        G::sync();
        const int n = mem.count;
        G::sync();
        if (n > KEEP) { lost = true; bound = ~0ull; bound_x = INFINITY; }   // not worth noting any more
        else if (n > KEEP / 4) {
          const u64 closer = tighten(mem.keep, n);
          if (closer > bound) { bound = closer; bound_x = value_of(bound); }
        }
      }
    }

    const float ctop = CAP ? cap.of(top) : top;
    if (__any_sync(0xffffffffu, !(ctop <= st.m))) {   // the warp's maximum has grown, or there is a NaN
      const Stat grown = {warp_max_nan(max_nan(ctop, st.m)), 0.f, 0.f};
      st = join(st, grown, scale);
    }
    if (top != -INFINITY) {
      bool one_by_one = !(st.m > DEEP) || flat; // all logits so far are at a type's lowest values, or NaN
      if (CAP && !one_by_one) {                 // or some, that are allowed, are not small against the cap
        one_by_one = !(top <= cap.most);
        float low = INFINITY;
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
          float x[N];
          Words<T>::unpack(cur[i], x);
#pragma unroll
          for (int k = 0; k < N; ++k) low = fminf(low, x[k]);
        }
        if (low < -cap.most) {
#pragma unroll
          for (int i = 0; i < BATCH; ++i) {
            float x[N];
            Words<T>::unpack(cur[i], x);
#pragma unroll
            for (int k = 0; k < N; ++k) one_by_one |= x[k] < -cap.most && x[k] > -INFINITY;
          }
        }
      }
      if (!one_by_one) {
        // a distance below FLOOR weighs nothing; raised to it, it is finite (-inf has one too, and so has the lowest logit under the highest reference)
        float2 z2 = make_float2(0.f, 0.f), s2 = make_float2(0.f, 0.f);
        const float2 m2 = make_float2(-st.m, -st.m), c2 = make_float2(scale, scale);
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
          float x[N];
          Words<T>::unpack(cur[i], x);
#pragma unroll
          for (int k = 0; k < N; k += 2) {
            const float y0 = CAP ? (x[k] == -INFINITY ? x[k] : cap.small(x[k])) : x[k], y1 = CAP ? (x[k + 1] == -INFINITY ? x[k + 1] : cap.small(x[k + 1])) : x[k + 1];
            const float2 far = __fadd2_rn(make_float2(y0, y1), m2), d = make_float2(max_nan(far.x, FLOOR), max_nan(far.y, FLOOR));
            const float2 t = __fmul2_rn(d, c2);
            const float2 e = make_float2(ex2(t.x), ex2(t.y));
            z2 = __fadd2_rn(z2, e);
            s2 = __ffma2_rn(e, d, s2);
          }
        }
        st.z += z2.x + z2.y;
        st.s += s2.x + s2.y;
      } else {
#pragma unroll 1
        for (int i = 0; i < BATCH * N; ++i) {
          const float x = Words<T>::at(reinterpret_cast<const T*>(&mem.word[slot + i / N][tid]), i % N);
          const float y = CAP ? cap.of(x) : x, d = y - st.m, e = ex2(d * scale);
          if (y != -INFINITY) { st.z += e; st.s += e == 0.f ? 0.f : e * d; }
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");

  // the team's sums, in a fixed order
  auto fold = [&]() {
    const Stat all = {warp_max_nan(st.m), 0.f, 0.f};
    st = join(st, all, scale);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { st.z += __shfl_xor_sync(0xffffffffu, st.z, o); st.s += __shfl_xor_sync(0xffffffffu, st.s, o); }
  };
  const Stat none = {-INFINITY, 0.f, 0.f};
  fold();
  if (NT > 32) {
    if (lane == 0) mem.part[warp] = st;
    G::sync();
    st = lane < NT / 32 ? mem.part[lane] : none;
    fold();
  }

  // the team's best keys, of single logits, over the rings
  u64* const single = reinterpret_cast<u64*>(&mem.word[0][0]);
  int n = 0;
  if (NT == 32 && exactly && want_top) {
    uint32_t img[WARP_ROW / 32];                             // of logits lane, lane + 32, ...; 0: behind the row
#pragma unroll
    for (int i = 0; i < WARP_ROW / 32; ++i) img[i] = i * 32 + lane < a.vocab ? image(Words<T>::at(row, i * 32 + lane)) : 0;
    uint32_t low = 1, high = 0xFFFFFFFFu;                    // at least top_k are at or above low
    for (int have = a.vocab; have > a.top_k && low < high;) {
      const uint32_t mid = low + (high - low) / 2 + 1;
      int c = 0;
#pragma unroll
      for (int i = 0; i < WARP_ROW / 32; ++i) c += img[i] >= mid;
      c = __reduce_add_sync(0xffffffffu, c);
      if (c >= a.top_k) { low = mid; have = c; }
      else high = mid - 1;
    }
    int more = 0;                                            // above low: all of them, so of low itself the rest, lowest ids first
#pragma unroll
    for (int i = 0; i < WARP_ROW / 32; ++i) more += img[i] > low;
    int equal = a.top_k - __reduce_add_sync(0xffffffffu, more);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < WARP_ROW / 32; ++i) {
      const unsigned same = __ballot_sync(0xffffffffu, img[i] == low);
      const bool take = img[i] > low || (img[i] == low && __popc(same & ((1u << lane) - 1)) < equal);
      const unsigned who = __ballot_sync(0xffffffffu, take);
      if (take) single[n + __popc(who & ((1u << lane) - 1))] = (u64)img[i] << 32 | (uint32_t)~(i * 32 + lane);
      n += __popc(who);
      equal = max(0, equal - __popc(same));
    }
    __syncwarp();
  } else if (want_top) {
    G::sync();
    int notes = mem.count;
    G::sync();
    lost |= notes > KEEP;
    if (!lost && notes > max(2 * a.top_k, NT / 4)) {         // (a bound takes as long as reading so many words at once)
      const u64 closer = tighten(mem.keep, notes);
      bound = closer > bound ? closer : bound;
      notes = mem.count;
    }
    lost |= notes * N > SINGLE;
    const int e_begin = max(0, w_begin * N - off), e_end = (int)min((long long)a.vocab, (long long)w_end * N - off);
    G::sync();
    if (tid == 0) mem.count = 0;
    G::sync();
    if (!lost) {
      for (int i0 = 0; i0 < notes * N; i0 += NT) {
        const int i = i0 + tid;
        u64 key = 0;
        if (i < notes * N) {
          const uint32_t word = (uint32_t)mem.keep[i / N];       // ~place
          const int id = (int)~word * N - off + i % N;
          if (id >= 0 && id < a.vocab) {
            key = key_of(Words<T>::at(row, id), id);
            if (((key >> 32) << 32 | word) < bound) key = 0;
          }
        }
        const int at = place_for(key != 0);
        if (key != 0) single[at] = key;
      }
    } else {
      u64 prefix = 0;
      int left = min(a.top_k, e_end - e_begin);
      for (int shift = 56; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += NT) mem.hist[i] = 0;
        G::sync();
        for (int i = e_begin + tid; i < e_end; i += NT) {
          const u64 key = key_of(Words<T>::at(row, i), i);
          if (shift == 56 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&mem.hist[(key >> shift) & 255], 1);
        }
        G::sync();
        int digit = 255;
        for (; digit > 0 && mem.hist[digit] < left; --digit) left -= mem.hist[digit];
        prefix |= (u64)digit << shift;
        G::sync();
      }
      for (int i = e_begin + tid; i < e_end; i += NT) {
        const u64 key = key_of(Words<T>::at(row, i), i);
        if (key >= prefix) single[atomicAdd(&mem.count, 1)] = key;
      }
    }
    G::sync();
    n = mem.count;
    G::sync();
    if (n > 64 + 2 * a.top_k) {                              // (or as counting over so many keys)
      tighten(single, n);
      n = mem.count;
    }
  }
  // a key's place is the number of larger ones
  auto place = [&](u64 key) {
    int above = 0;
#pragma unroll 4
    for (int j = 0; j < n; ++j) above += single[j] > key;
    return above;
  };

  if (NT > 32 && blocks > 1) {    // the first block takes the others' sums and keys
    if (tid == 0) mem.stat = st;
    for (int i = tid; i < a.top_k; i += NT) mem.best[i] = 0;
    G::sync();
    for (int i = tid; i < n; i += NT) {
      const u64 key = single[i];
      const int above = place(key);
      if (above < a.top_k) mem.best[above] = key;
    }
    cluster_sync();
    if (rank == 0) {
      st = lane < blocks ? *in_block(&mem.stat, min(lane, blocks - 1)) : none;
      fold();
      n = want_top ? blocks * a.top_k : 0;
      for (int i = tid; i < n; i += NT) single[i] = in_block(&mem.best[0], i / a.top_k)[i % a.top_k];
    }
    cluster_sync();               // nobody leaves before it has been read
    if (rank != 0) return;
  }
  if (NT > 32) G::sync();

  const float logz = logf(st.z);
  auto logp = [&](float x) {
    if (x == -INFINITY) return -INFINITY;
    return ((CAP ? cap.of(x) : x) - st.m) / a.temperature - logz;
  };
  if (a.entropy_out && tid == 0) a.entropy_out[r] = st.z == 0.f ? 0.f : logz - st.s / st.z / a.temperature;
  if (a.given_out)
    for (int i = tid; i < a.num_given; i += NT) {
      const long long id = i == tid ? given_id : a.given[(long long)r * a.num_given + i];
      a.given_out[(long long)r * a.num_given + i] = id < 0 || id >= a.vocab ? 0.f : logp(i == tid ? given_x : Words<T>::at(row, id));
    }
  for (int i = tid; i < n; i += NT) {
    const u64 key = single[i];
    const int above = key == 0 ? a.top_k : place(key);
    if (above >= a.top_k) continue;
    if (a.top_ids_out) a.top_ids_out[(long long)r * a.top_k + above] = (int)~(uint32_t)key;
    if (a.top_out) a.top_out[(long long)r * a.top_k + above] = logp(value_of(key));
  }
}

template <typename T, int NT, bool CAP>
cudaError_t logprobs_launch(const phx_logprobs_args& a, int blocks, cudaStream_t stream) {
  constexpr int smem = (NT == 32 ? WARP_ROWS : 1) * (int)sizeof(typename Shape<NT>::Memory);
  static SmemLimit limit;
  const cudaError_t e = smem > 48 * 1024 ? limit.raise(logprobs_kernel<T, NT, CAP>, smem) : cudaSuccess;
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t lc;
  memset(&lc, 0, sizeof(lc));
  lc.gridDim = dim3((unsigned)(NT == 32 ? (a.rows + WARP_ROWS - 1) / WARP_ROWS : a.rows * blocks));
  lc.blockDim = dim3(NT == 32 ? 32 * WARP_ROWS : NT);
  lc.dynamicSmemBytes = smem; lc.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)blocks; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
  lc.attrs = at; lc.numAttrs = 1;
  return cudaLaunchKernelEx(&lc, logprobs_kernel<T, NT, CAP>, a, blocks);
}
// Threads of a row: enough for its words in one batch, up to the row's part of the device's (148 SMs of 1024 threads at this kernel's registers), rounded up to
// what there is: a warp for rows it can hold, else a block of 256, of 1024, else a cluster of up to eight of those.  Rounding up makes 149 to 295 long rows two rounds of blocks (148
// fp32 rows of 131072 with best 8 take 23 us, 149 take 41, 296 take 40), 75 to 147 pairs that do not all fit (74 rows 18 us, 75 rows 30).
template <typename T, bool CAP>
cudaError_t logprobs_dispatch(const phx_logprobs_args& a, cudaStream_t stream) {
  const long long need = (a.vocab + 2ll * Words<T>::N) / (Words<T>::N * 4) + 1;
  const long long room = (long long)device_sms() * 1024 / a.rows;
  const long long threads = need < room ? need : room;
  if (a.vocab <= WARP_ROW) return logprobs_launch<T, 32, CAP>(a, 1, stream);
  if (threads <= 512 || a.rows > 1 << 27) return logprobs_launch<T, 256, CAP>(a, 1, stream);
  const int blocks = threads <= 1024 ? 1 : threads <= 2048 ? 2 : threads <= 4096 ? 4 : 8;
  return logprobs_launch<T, 1024, CAP>(a, blocks, stream);
}

}  // namespace
}  // namespace phx

using namespace phx;

extern "C" phx_status phx_token_logprobs_device(int32_t device, const phx_logprobs_args* args, void* stream) {
  auto bad = [](const char* m) { set_global_error(std::string("phx_token_logprobs_device: ") + m); return PHX_E_ARG; };
  if (!args) return bad("null argument");
  const phx_logprobs_args& a = *args;
  if (a.rows < 0 || a.vocab < 1 || a.num_given < 0) return bad("rows and num_given must not be negative, vocab positive");
  if (a.vocab > 1 << 28) return bad("vocab must be at most 2^28");
  if (a.top_k < 0 || a.top_k > PHX_LOGPROBS_MAX_TOP || a.top_k > a.vocab) return bad("top_k must be at most 128 and at most vocab");
  if (!(a.temperature > 0.f) || isinf(a.temperature)) return bad("temperature must be positive");
  if (!(a.cap == a.cap) || isinf(a.cap)) return bad("cap must be finite");
  if (a.stride < a.vocab) return bad("stride must cover a row");
  if (a.is_bf16 != 0 && a.is_bf16 != 1) return bad("is_bf16 must be 0 or 1");
  if (a.rows == 0) return PHX_OK;
  if (!a.logits || (reinterpret_cast<uintptr_t>(a.logits) & (a.is_bf16 ? 1 : 3)) != 0) return bad("logits must be a buffer of whole elements");
  if (a.num_given > 0 && a.given_out && !a.given) return bad("given is required with given_out");
  DeviceScope scope(device);
  if (!scope.ok()) { set_global_error("phx_token_logprobs_device: cudaSetDevice failed"); return PHX_E_CUDA; }
  cudaStream_t st = (cudaStream_t)stream;
  const cudaError_t e = taken_back(a.is_bf16 ? (a.cap > 0.f ? logprobs_dispatch<bf16, true>(a, st) : logprobs_dispatch<bf16, false>(a, st))
                                             : (a.cap > 0.f ? logprobs_dispatch<float, true>(a, st) : logprobs_dispatch<float, false>(a, st)));
  if (e != cudaSuccess) { set_global_error(std::string("phx_token_logprobs_device: ") + cudaGetErrorString(e)); return PHX_E_CUDA; }
  dispatch_note(DK_TOKEN_LOGPROBS);
  return PHX_OK;
}
