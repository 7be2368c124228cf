// Eviction from a paged cache by the weights that its keys received (phx_evict_device): per request and key head the first keys, the last ones and the heaviest
// of the others stay, at most `budget` of them, and move together in their order, in place.
//
// Two launches.  evict_select_kernel finds what stays: a cluster of blocks shares a head's keys, each with its stretch of weights in shared memory as integers of the
// same order, and the smallest weight that stays comes out of three histograms, of 11, 11 and 10 bits, summed over the cluster (fewer where a digit decides already);
// the places that stay are then numbered by prefix sums, equal weights by their order.  evict_move_kernel moves rows: a block takes what goes to one chunk of a head's places,
// keys, values and weights, into shared memory, says so, and writes it once what it writes over has been read.  A row only ever moves to the front, so what lies in a chunk's
// places is taken by that chunk or one before it, by two at most: it is no more than fills one.  Chunks are handed out in order, by a counter, so a block only waits for blocks that
// have begun, and whose reads wait for nothing.
// Measured (us, keys that leave for the first time, cold caches): 64 x 4 heads of up to 4096 keys of 128, half of them stay (375 k rows change their place, 387 MB read and written): select 19, move 66 =
// 5.9 TB/s, the call 88; 2 x 4 heads of 100 k keys, a third stays: 25 and 55 (262 k rows, 270 MB, 4.9 TB/s, by 3280 blocks that wait for one another's reads), the call 84.  With a wait for all chunks in front the second took 73 for its move where 61 were left with two; blocks that went through a head's places from front to
// back by themselves took 247 for the second and 89 for the first.
#include <string>

#include "cache_batch.cuh"
#include "sm100_ptx.cuh"

namespace phx {
namespace {

using namespace sm100;

constexpr int MOST_BUDGET = 1 << 30;   // the kernels count past it by a grid's threads, in 32 bits

struct EvictView {
  phx_cache_batch c;
  phx_evict_args a;
  uint64_t page_magic;           // ceil(2^36 / (page_size / 16))
  int held;                      // weights that a block of the select keeps in shared memory
  int rows;                      // places of a chunk
  int chunks;                    // of a head
  int alone;                     // few rows: the select's blocks move them, too
  int* ticket;                   // the next chunk to hand out
  int* read;                     // [batch][heads][chunks] whether it has been read
};
// x / page_size for x below 2^31: exact, as x / 16 < 2^27 and page_size / 16 <= 256 (the product's error stays below 2^27 * 256 < 2^36)
__device__ __forceinline__ int page_column(const EvictView& t, int x) { return (int)(((uint64_t)((uint32_t)x >> 4) * t.page_magic) >> 36); }

struct EvictRequest { int length, sinks, behind; bool ok; };   // of a request over its budget: [sinks, behind) is what some of leaves
__device__ __forceinline__ EvictRequest evict_request(const EvictView& t, int b) {
  EvictRequest r;
  const int len = t.c.lengths[b];
  r.ok = len >= 0 && len <= cache_columns(t.c);
  r.length = max(0, (int)min((long long)len, cache_columns(t.c)));
  r.sinks = min(t.a.sinks, r.length); r.behind = r.length - min(t.a.recent, r.length);
  return r;
}

// ---- a chunk of a head's places, moved by a block ------------------------------------------------------------------------------

// Of each place: its key's row of the pool and that which it receives (-1: none), its word among the weights, the weight that it receives
struct ChunkPlaces { int to[256], from[256], word[256]; float weight[256]; };
template <int THREADS>
struct ChunkMove {
  const EvictView& t;
  ChunkPlaces& at;
  uint8_t* data;                                             // rows of keys, behind them rows of values
  int b, h, first, count, pieces;                            // pieces of 16 bytes in a row
  __device__ __forceinline__ bool good(int page) const {
    if ((unsigned)page < (unsigned)t.c.num_pages) return true;
    cache_report(t.c, CACHE_BAD_PAGE);
    return false;
  }
  // place `i` of the chunk, in page `to`, receives place `src`, in `page`; whether it is another
  __device__ __forceinline__ bool place(int i, int src, int to, int page) {
    const int from_slot = src - page_column(t, src) * t.c.page_size, to_slot = first + i - page_column(t, first + i) * t.c.page_size;
    const bool there = good(to), moves = good(page) && there && src != first + i;
    at.from[i] = moves ? (page * 2 * t.c.num_kv_heads + h) * t.c.page_size + from_slot : -1;   // the pool's rows fit 31 bits
    at.to[i] = (to * 2 * t.c.num_kv_heads + h) * t.c.page_size + to_slot;
    at.word[i] = (to * t.c.num_kv_heads + h) * t.c.page_size + to_slot;
    if (moves)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(at.weight + i)), "l"(t.a.weights + ((long long)page * t.c.num_kv_heads + h) * t.c.page_size + from_slot) : "memory");
    return moves;
  }
  // A thread has one piece of every so many rows, of the key and the value.  (With addresses worked out a piece at a time the move was issue-bound: 64 x 4 heads 82 us, 2 x 4 long ones 62.)
  __device__ __forceinline__ void fetch() {                  // behind a barrier behind place()
    const int row_of = threadIdx.x / pieces, piece = threadIdx.x - row_of * pieces, row_bytes = pieces * 16;
    const uint16_t* const keys = t.c.pages + piece * 8;
    const uint16_t* const values = keys + (long long)t.c.num_kv_heads * t.c.page_size * t.c.key_size;
    const uint32_t to = smem_u32(data) + piece * 16;
#pragma unroll 4
    for (int i = row_of; i < count; i += THREADS / pieces) {
      const int row = at.from[i];
      if (row < 0) continue;
      const long long from = (long long)row * t.c.key_size;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + i * row_bytes), "l"(keys + from) : "memory");
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + (count + i) * row_bytes), "l"(values + from) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  __device__ __forceinline__ void store() const {            // once nothing reads what it writes over
    const int row_of = threadIdx.x / pieces, piece = threadIdx.x - row_of * pieces, row_bytes = pieces * 16;
    uint16_t* const keys = t.c.pages + piece * 8;
    uint16_t* const values = keys + (long long)t.c.num_kv_heads * t.c.page_size * t.c.key_size;
    const uint8_t* const from = data + piece * 16;
#pragma unroll 4
    for (int i = row_of; i < count; i += THREADS / pieces) {
      if (at.from[i] < 0) continue;
      const long long to = (long long)at.to[i] * t.c.key_size;
      *reinterpret_cast<uint4*>(keys + to) = *reinterpret_cast<const uint4*>(from + i * row_bytes);
      *reinterpret_cast<uint4*>(values + to) = *reinterpret_cast<const uint4*>(from + (count + i) * row_bytes);
    }
    for (int i = threadIdx.x; i < count; i += THREADS)
      if (at.from[i] >= 0) t.a.weights[at.word[i]] = at.weight[i];
  }
};

// ---- what stays ------------------------------------------------------------------------------------------------------------

constexpr int SEL_THREADS = 1024, SEL_FEW = 256, SEL_BINS = 2048, SEL_COARSE = SEL_BINS / 32, SEL_RANKS = 8;
struct alignas(16) SelectSmem {
  uint32_t hist[3][SEL_BINS];
  uint32_t coarse[3][SEL_COARSE];        // sums of 32 bins
  uint32_t warp_more[SEL_THREADS / 32], warp_same[SEL_THREADS / 32];
  uint32_t taken[2];                     // this block's heavier weights, and those equal to the smallest that stays
  uint32_t bin, above, in_bin;
};

static_assert(sizeof(SelectSmem) % 16 == 0 && sizeof(ChunkPlaces) % 16 == 0, "what lies behind them is copied to in pieces of 16 bytes");

// the order of weights as that of unsigned integers: NaN above all, zeros alike
__device__ __forceinline__ uint32_t weight_order(float w) {
  uint32_t u = __float_as_uint(w);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if (u == 0x80000000u) u = 0;
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint32_t remote_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
template <int THREADS>
__global__ void __launch_bounds__(THREADS) evict_select_kernel(const EvictView t) {
  constexpr int WARPS = THREADS / 32;
  extern __shared__ __align__(16) uint8_t smem_bytes[];
  SelectSmem& sm = *reinterpret_cast<SelectSmem*>(smem_bytes);
  uint32_t* const held = reinterpret_cast<uint32_t*>(smem_bytes + sizeof(SelectSmem));
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, h = blockIdx.y, b = blockIdx.z, rank = blockIdx.x, ranks = gridDim.x;
  const EvictRequest rq = evict_request(t, b);
  if (rank == 0 && h == 0 && tid == 0 && !rq.ok) cache_report(t.c, CACHE_BAD_OFFSETS);
  int* const kept = t.a.kept_out + ((long long)b * t.c.num_kv_heads + h) * t.a.budget;
  if (t.alone && rank == 0 && h == 0 && tid == 0) t.a.lengths_out[b] = min(rq.length, t.a.budget);
  if (!t.alone && rank == 0) {                               // for the launch behind
    int* const read = t.read + ((long long)b * t.c.num_kv_heads + h) * t.chunks;
    for (int i = tid; i < t.chunks; i += THREADS) read[i] = 0;
    if (b == 0 && h == 0 && tid == 0) *t.ticket = 0;
  }
  if (rq.length <= t.a.budget) {                             // the same for the whole cluster
    for (int i = rank * THREADS + tid; i < t.a.budget; i += ranks * THREADS) kept[i] = i < rq.length ? i : -1;
    return;
  }
  const int* const table = t.c.block_table + (long long)b * t.c.table_stride;
  const int middle = rq.behind - rq.sinks, per = (middle + ranks - 1) / ranks, from = rq.sinks + min(rank * per, middle), count = min(per, rq.behind - from);
  auto weight_at = [&](int key) {
    const int col = page_column(t, key), page = table[col];
    if ((unsigned)page >= (unsigned)t.c.num_pages) { cache_report(t.c, CACHE_BAD_PAGE); return 0u; }
    return weight_order(t.a.weights[((long long)page * t.c.num_kv_heads + h) * t.c.page_size + key - col * t.c.page_size]);
  };
  const bool in_smem = per <= t.held;
  for (int i = tid; i < 3 * SEL_BINS; i += THREADS) (&sm.hist[0][0])[i] = 0;
  if (in_smem) {                                             // loads without a condition: a batch of pages, then of weights, on their way at once
    constexpr int BATCH = 4;
    for (int i0 = tid; i0 < count; i0 += BATCH * THREADS) {
      int page[BATCH], slot[BATCH];
      float w[BATCH];
      bool bad = false;
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        const int key = from + min(i0 + k * THREADS, count - 1), col = page_column(t, key);
        page[k] = table[col]; slot[k] = key - col * t.c.page_size;
      }
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        const bool good = (unsigned)page[k] < (unsigned)t.c.num_pages;
        bad |= !good;
        w[k] = t.a.weights[((long long)(good ? page[k] : 0) * t.c.num_kv_heads + h) * t.c.page_size + slot[k]];
        page[k] = good;
      }
#pragma unroll
      for (int k = 0; k < BATCH; ++k) if (i0 + k * THREADS < count) held[i0 + k * THREADS] = page[k] ? weight_order(w[k]) : 0u;
      if (bad) cache_report(t.c, CACHE_BAD_PAGE);
    }
  }
  __syncthreads();
  auto order_at = [&](int i) { return in_smem ? held[i] : weight_at(from + i); };

  // the smallest order that stays, and how many of those equal to it
  uint32_t least = 0xffffffffu, equal = 0, prefix = 0;
  uint32_t want = (uint32_t)(t.a.budget - rq.sinks - (rq.length - rq.behind));
#pragma unroll 1
  for (int pass = 0; pass < 3 && want > 0; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    uint32_t* const hist = sm.hist[pass];
    for (int i = tid; i < count; i += THREADS) {
      const uint32_t v = order_at(i);
      if (pass == 0 || (v >> (shift + bits)) == prefix) atomicAdd(&hist[(v >> shift) & ((1u << bits) - 1)], 1u);
    }
    __syncthreads();
    for (int c = warp; c < SEL_COARSE; c += WARPS) {
      const uint32_t sum = __reduce_add_sync(0xffffffffu, hist[c * 32 + lane]);
      if (lane == 0) sm.coarse[pass][c] = sum;
    }
    if (ranks > 1) cluster_sync_all(); else __syncthreads();
    if (warp == 0) {                                         // the bin of the last that stays, from the top: among the coarse ones first
      auto sum_of = [&](const uint32_t* p) {
        if (ranks == 1) return *p;
        uint32_t v[SEL_RANKS], sum = 0;
        const uint32_t addr = smem_u32(p);
#pragma unroll
        for (int r = 0; r < SEL_RANKS; ++r) v[r] = r < ranks ? remote_u32(mapa_shared(addr, r)) : 0;
#pragma unroll
        for (int r = 0; r < SEL_RANKS; ++r) sum += v[r];
        return sum;
      };
      auto upto = [&](uint32_t v) {                          // with those of the lanes in front
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const uint32_t x = __shfl_up_sync(0xffffffffu, v, o); v += lane >= o ? x : 0; }
        return v;
      };
      const int c0 = SEL_COARSE - 1 - 2 * lane;              // this lane's coarse bins: c0, c0 - 1
      const uint32_t s0 = sum_of(&sm.coarse[pass][c0]), s1 = sum_of(&sm.coarse[pass][c0 - 1]), with = upto(s0 + s1), front = with - s0 - s1;
      const int owner = __ffs(__ballot_sync(0xffffffffu, with >= want)) - 1;
      const bool second = front + s0 < want;
      const int coarse = __shfl_sync(0xffffffffu, second ? c0 - 1 : c0, owner);
      const uint32_t above = __shfl_sync(0xffffffffu, second ? front + s0 : front, owner);
      const uint32_t mine = sum_of(&hist[coarse * 32 + 31 - lane]), to = above + upto(mine);
      const int at = __ffs(__ballot_sync(0xffffffffu, to >= want)) - 1;
      if (lane == at) { sm.bin = (uint32_t)(coarse * 32 + 31 - lane); sm.above = to - mine; sm.in_bin = mine; }
    }
    __syncthreads();
    prefix = (prefix << bits) | sm.bin;
    want -= sm.above;
    least = prefix << shift; equal = want;                   // of the last pass: the order itself
    if (sm.in_bin == want) { least -= 1; equal = 0; break; } // the whole bin stays (never the lowest bin of all: more keys than stay)
    __syncthreads();
  }

  // numbers of what stays: a warp's keys lie one behind the other, 32 at a time
  const int seg = ((count + WARPS - 1) / WARPS + 31) & ~31, i0 = min(warp * seg, count), i1 = min(i0 + seg, count);
  uint32_t more = 0, same = 0;
  for (int i = i0 + lane; i - lane < i1; i += 32) {
    const uint32_t v = i < i1 ? order_at(i) : 0;
    more += __popc(__ballot_sync(0xffffffffu, i < i1 && v > least)); same += __popc(__ballot_sync(0xffffffffu, i < i1 && v == least));
  }
  if (lane == 0) { sm.warp_more[warp] = more; sm.warp_same[warp] = same; }
  __syncthreads();
  uint32_t more_before = __reduce_add_sync(0xffffffffu, lane < warp ? sm.warp_more[lane] : 0), same_before = __reduce_add_sync(0xffffffffu, lane < warp ? sm.warp_same[lane] : 0);
  if (ranks > 1) {
    if (tid == THREADS - 32) { sm.taken[0] = more_before + more; sm.taken[1] = same_before + same; }   // the last warp
    cluster_sync_all();
    const bool in_front = lane < rank;
    more_before += __reduce_add_sync(0xffffffffu, in_front ? remote_u32(mapa_shared(smem_u32(&sm.taken[0]), in_front ? lane : 0)) : 0);
    same_before += __reduce_add_sync(0xffffffffu, in_front ? remote_u32(mapa_shared(smem_u32(&sm.taken[1]), in_front ? lane : 0)) : 0);
  }
  for (int i = i0 + lane; i - lane < i1; i += 32) {
    const uint32_t v = i < i1 ? order_at(i) : 0, in_front = (1u << lane) - 1;
    const bool heavier = i < i1 && v > least, like = i < i1 && v == least;
    const uint32_t heavier_of = __ballot_sync(0xffffffffu, heavier), like_of = __ballot_sync(0xffffffffu, like);
    const uint32_t likes = same_before + __popc(like_of & in_front), to = rq.sinks + more_before + __popc(heavier_of & in_front) + min(likes, equal);
    if ((heavier || (like && likes < equal)) && to < (uint32_t)t.a.budget) kept[to] = from + i;
    more_before += __popc(heavier_of); same_before += __popc(like_of);
  }
  // the first keys and the last ones
  const int recent = rq.length - rq.behind;
  for (int i = rank * THREADS + tid; i < rq.sinks; i += ranks * THREADS) kept[i] = i;
  for (int i = rank * THREADS + tid; i < recent; i += ranks * THREADS) kept[t.a.budget - recent + i] = rq.behind + i;
  if (ranks > 1) cluster_sync_all();                         // the others may still be reading this block's counts; the places that they wrote are there
  if (!t.alone || rank > 0) return;
  __syncthreads();
  if (kept[t.a.budget - 1] < t.a.budget) return;
  ChunkMove<THREADS> move{t, *reinterpret_cast<ChunkPlaces*>(held), reinterpret_cast<uint8_t*>(held) + sizeof(ChunkPlaces), b, h, 0, t.a.budget, t.c.key_size / 8};
  for (int i = tid; i < t.a.budget; i += THREADS) move.place(i, kept[i], table[page_column(t, i)], table[page_column(t, kept[i])]);
  __syncthreads();
  move.fetch();
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  move.store();
}

// ---- moving together ---------------------------------------------------------------------------------------------------------

// Bytes of a chunk's keys and values: 16, 24, 32, 40 KB, of rows of 128, 64 x 4 heads of 4096 keys 90, 82, 80, 80 us, 2 x 4 of 100 k 89, 88, 83, 81 (with the select)
constexpr int MOVE_THREADS = 256, MOVE_BYTES = 40 * 1024;

// Bounded wait until the n words at p are set, by all threads; false when the limit ran out or another wait's did.  Every thread comes out with the same answer.
__device__ __forceinline__ bool wait_all_set(const int* p, int n, volatile int* status) {
  unsigned long long t0 = 0;
  for (uint32_t it = 0;; ++it) {
    bool all = true, over = false;
    for (int i = threadIdx.x; i < n; i += MOVE_THREADS) {
      int v;
      asm volatile("ld.acquire.gpu.global.b32 %0, [%1];" : "=r"(v) : "l"(p + i) : "memory");
      all &= v != 0;
    }
    if ((it & 0xff) == 0xff && threadIdx.x == 0) {
      const unsigned long long now = globaltimer_ns();
      if (t0 == 0) t0 = now;
      const unsigned us = (unsigned)status[1];
      over = status[0] != 0 || now - t0 > (us ? 1000ull * us : WAIT_LIMIT_NS);
    }
    if (__syncthreads_and(all)) return true;
    if (__syncthreads_or(over)) { if (threadIdx.x == 0) status[0] = 1; return false; }
  }
}

__global__ void __launch_bounds__(MOVE_THREADS) evict_move_kernel(const EvictView t) {
  __shared__ __align__(16) uint8_t data[MOVE_BYTES];
  __shared__ ChunkPlaces places;
  __shared__ int ticket;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int tid = threadIdx.x, heads = t.c.batch * t.c.num_kv_heads;
  if (tid == 0) ticket = atomicAdd(t.ticket, 1);
  __syncthreads();
  const int chunk = ticket / heads, of = ticket - chunk * heads, b = of / t.c.num_kv_heads, h = of - b * t.c.num_kv_heads;
  const int* const kept = t.a.kept_out + (long long)of * t.a.budget;
  // the one reader of this request's length in this launch, so that lengths_out may be lengths
  if (chunk == 0 && h == 0 && tid == 0) t.a.lengths_out[b] = min(evict_request(t, b).length, t.a.budget);
  const int first = chunk * t.rows, count = min(t.rows, t.a.budget - first);
  const int* const table = t.c.block_table + (long long)b * t.c.table_stride;
  ChunkMove<MOVE_THREADS> move{t, places, data, b, h, first, count, t.c.key_size / 8};
  // Round trips: the place that this thread's place receives and its page at once (the first `budget` places have columns where a request is over its budget), that one's page, its rows.
  const int last = kept[t.a.budget - 1];
  int src = -1, to = -1;
  const int col = page_column(t, first + tid);
  if (tid < count) {
    src = kept[first + tid];
    if (col < t.c.table_cols) to = table[col];
  }
  if (last < t.a.budget) return;                             // at most `budget` keys: all where they are
  int* const read = t.read + (long long)of * t.chunks;
  if (!__syncthreads_or(tid < count && move.place(tid, src, to, table[page_column(t, src)]))) {   // all stays where it is
    if (tid == 0) asm volatile("st.release.gpu.global.b32 [%0], %1;" ::"l"(read + chunk), "r"(1) : "memory");
    return;
  }
  move.fetch();
  // under the copies: the first of the kept rows that lies in this chunk's places (or behind), 256 looked at at a time
  int reader = 0;
  for (int left = first + 1; left > 0;) {                    // it is not behind place `first` of the kept ones
    const int step = (left + MOVE_THREADS - 1) / MOVE_THREADS, at = tid * step;
    const int before = __syncthreads_count(at < left && kept[reader + min(at, left - 1)] < first);
    if (before == 0) break;
    reader += (before - 1) * step + 1;
    left = min(step - 1, left - (before - 1) * step - 1);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  if (tid == 0) asm volatile("st.release.gpu.global.b32 [%0], %1;" ::"l"(read + chunk), "r"(1) : "memory");
  const int from_chunk = reader / t.rows, to_chunk = min(chunk, (reader + t.rows - 1) / t.rows + 1);   // in front of this one: whose sources may lie here
  if (!wait_all_set(read + from_chunk, to_chunk - from_chunk, t.c.status_dev)) return;
  move.store();
}

}  // namespace
}  // namespace phx

using namespace phx;

extern "C" phx_status phx_evict_device(int32_t device, const phx_cache_batch* cache, const phx_evict_args* args, void* stream) {
  auto bad = [](const char* m) { set_global_error(std::string("phx_evict_device: ") + m); return PHX_E_ARG; };
  EvictView t;
  if (!cache || !args) return bad("null argument");
  t.c = *cache; t.a = *args;
  t.c.q_start = t.c.lengths; t.c.num_tokens = 1;               // not used here: what cache_check asks for
  const char* what = cache_check(&t.c);
  if (*what) return bad(what);
  if (t.c.batch > 65535) return bad("at most 65535 requests");
  if (t.a.budget < 1 || t.a.sinks < 0 || t.a.recent < 0 || (long long)t.a.sinks + t.a.recent > t.a.budget) return bad("budget must be at least 1 and hold sinks + recent keys");
  if (t.a.budget > MOST_BUDGET) return bad("budget must be at most 2^30");
  if (t.a.max_keys < 0) return bad("negative size");
  if (t.c.batch == 0) return PHX_OK;
  if (t.c.num_pages == 0) return bad("an empty pool has no keys");
  if (!t.a.weights || !t.a.lengths_out || !t.a.kept_out) return bad("weights, lengths_out and kept_out are required");
  const long long columns = (long long)t.c.table_cols * t.c.page_size;
  if (t.a.max_keys > columns) t.a.max_keys = columns;
  const int e = t.c.page_size / 16;
  t.page_magic = ((1ull << 36) + e - 1) / e;
  const long long heads = (long long)t.c.batch * t.c.num_kv_heads;
  t.rows = MOVE_BYTES / (4 * t.c.key_size);                   // 80, 160,
  if (t.rows > MOVE_THREADS) t.rows = MOVE_THREADS;           // and of heads of 32 one a thread
  t.chunks = (int)(((long long)t.a.budget + t.rows - 1) / t.rows);
  if (heads * t.chunks > 2147483647ll) return bad("budget x heads x batch is too large");
  if (t.a.workspace_bytes < 16 + heads * t.chunks * 4) return bad("workspace is smaller than phx_tree_workspace_bytes or too small for this many heads and budget");
  if (!t.a.workspace || !aligned16(t.a.workspace)) return bad("workspace must be a 16-byte aligned buffer");
  t.ticket = static_cast<int*>(t.a.workspace);
  t.read = t.ticket + 4;
  DeviceScope scope(device);
  if (!scope.ok()) { set_global_error("phx_evict_device: cudaSetDevice failed"); return PHX_E_CUDA; }
  cudaStream_t st = (cudaStream_t)stream;

  // Blocks of a cluster: as long as the heads' clusters fit the device twice over and a block keeps 1024 weights
  int ranks = 1;
  while (ranks < SEL_RANKS && heads * ranks * 2 <= 2ll * device_sms() && t.a.max_keys / ranks > 1024) ranks *= 2;
  constexpr int MOST_HELD = 48 * 1024;                        // weights: 192 KB beside the histograms; longer stretches are read from memory at each pass
  const long long per = (t.a.max_keys + ranks - 1) / ranks;
  t.held = (int)(per < MOST_HELD ? per : MOST_HELD);
  // Up to 256 rows and 64 KB of keys and values a head, the select's block moves them itself, in shared memory that the weights were in: a launch less.  Its heads may not all have read
  // a length that is written over, so lengths_out must not be lengths.
  const long long move_bytes = (long long)sizeof(ChunkPlaces) + (long long)t.a.budget * 4 * t.c.key_size;
  t.alone = t.a.budget <= 256 && move_bytes <= 68 * 1024 && (t.a.lengths_out + t.c.batch <= t.c.lengths || t.c.lengths + t.c.batch <= t.a.lengths_out);
  if (t.alone && t.held * 4 < move_bytes) t.held = (int)((move_bytes + 3) / 4);
  // More blocks than SMs, of up to 4096 keys each: small ones, four or five an SM (832 heads of 67 keys: 15 us, 40 by blocks of 1024; 1024 of 3000: 134 and 157, with the
  // move; 512 of 8000: 246 and 241, of 20 k: 431 and 403; 32 of 300 alike)
  const bool few = heads * ranks > device_sms() && per <= 4096;
  const int select_smem = (int)sizeof(SelectSmem) + t.held * 4;
  static SmemLimit select_limit, few_limit;
  std::string err;
  auto launch = [&]() -> phx_status {
    PHX_CUDA_TRY(select_limit.raise(evict_select_kernel<SEL_THREADS>, (int)sizeof(SelectSmem) + MOST_HELD * 4), err);
    PHX_CUDA_TRY(few_limit.raise(evict_select_kernel<SEL_FEW>, (int)sizeof(SelectSmem) + MOST_HELD * 4), err);
    cudaLaunchConfig_t lc;
    memset(&lc, 0, sizeof(lc));
    lc.gridDim = dim3(ranks, t.c.num_kv_heads, t.c.batch); lc.blockDim = dim3(few ? SEL_FEW : SEL_THREADS); lc.dynamicSmemBytes = select_smem; lc.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ranks; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    lc.attrs = at; lc.numAttrs = 1;
    PHX_CUDA_TRY(few ? cudaLaunchKernelEx(&lc, evict_select_kernel<SEL_FEW>, t) : cudaLaunchKernelEx(&lc, evict_select_kernel<SEL_THREADS>, t), err);
    if (!t.alone) PHX_CUDA_TRY(launch_programmatic(evict_move_kernel, dim3((unsigned)(heads * t.chunks)), dim3(MOVE_THREADS), 0, st, t), err);
    dispatch_note(DK_CACHE_EVICT);
    return PHX_OK;
  };
  const phx_status s = launch();
  if (s != PHX_OK) {
    (void)cudaGetLastError();
    set_global_error("phx_evict_device: " + err);
  }
  return s;
}
