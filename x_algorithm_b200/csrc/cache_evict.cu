// Eviction from a paged cache by the weights that its keys received (phx_evict_device): per request and key head the first keys, the last ones and the heaviest
// of the others stay, at most `budget` of them, and move together in their order, in place.
//
// Two launches.  evict_select_kernel finds what stays: a cluster of blocks shares a head's keys, each with its stretch of weights in shared memory as integers of the
// same order, and the smallest weight that stays comes out of three histograms, of 11, 11 and 10 bits, summed over the cluster (fewer where a digit decides already);
// the places that stay are then numbered by prefix sums, equal weights by their order.  evict_move_kernel moves rows: a block takes the keys or the values (or some of
// their columns, or the weights) of one head from the front to the back.  A row only ever moves forward, so what a chunk of places receives lies in it or behind:
// once a block has read a chunk and all before it, it may write there, and later chunks may be on their way meanwhile.  No block waits for another.
#include <string>

#include "cache_batch.cuh"
#include "sm100_ptx.cuh"

namespace phx {
namespace {

using namespace sm100;

struct EvictView {
  phx_cache_batch c;
  phx_evict_args a;
  uint64_t page_magic;           // ceil(2^36 / (page_size / 16))
  int held;                      // weights that a block of the select keeps in shared memory
  int slices;                    // blocks that share a head's rows by columns
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

// ---- what stays ------------------------------------------------------------------------------------------------------------

constexpr int SEL_THREADS = 512, SEL_BINS = 2048;
struct SelectSmem {
  uint32_t hist[3][SEL_BINS];
  uint32_t warp_sum[2][SEL_THREADS / 32];
  uint32_t taken[2];             // this block's heavier weights, and those equal to the smallest that stays
  uint32_t bin, above, in_bin;
};

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
__device__ __forceinline__ uint4 remote_u32x4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}

__global__ void __launch_bounds__(SEL_THREADS) evict_select_kernel(const EvictView t) {
  extern __shared__ __align__(16) uint8_t smem_bytes[];
  SelectSmem& sm = *reinterpret_cast<SelectSmem*>(smem_bytes);
  uint32_t* const held = reinterpret_cast<uint32_t*>(smem_bytes + sizeof(SelectSmem));
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, h = blockIdx.y, b = blockIdx.z, rank = blockIdx.x, ranks = gridDim.x;
  const EvictRequest rq = evict_request(t, b);
  if (rank == 0 && h == 0 && tid == 0 && !rq.ok) cache_report(t.c, CACHE_BAD_OFFSETS);
  int* const kept = t.a.kept_out + ((long long)b * t.c.num_kv_heads + h) * t.a.budget;
  if (rq.length <= t.a.budget) {                             // the same for the whole cluster
    for (int i = rank * SEL_THREADS + tid; i < t.a.budget; i += ranks * SEL_THREADS) kept[i] = i < rq.length ? i : -1;
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
  for (int i = tid; i < 3 * SEL_BINS; i += SEL_THREADS) (&sm.hist[0][0])[i] = 0;
  if (in_smem) {
#pragma unroll 4
    for (int i = tid; i < count; i += SEL_THREADS) held[i] = weight_at(from + i);
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
    for (int i = tid; i < count; i += SEL_THREADS) {
      const uint32_t v = order_at(i);
      if (pass == 0 || (v >> (shift + bits)) == prefix) atomicAdd(&hist[(v >> shift) & ((1u << bits) - 1)], 1u);
    }
    if (ranks > 1) cluster_sync_all(); else __syncthreads();
    // bins 4 tid' .. 4 tid' + 3, from the top: tid 0 has the highest
    const int bin0 = SEL_BINS - 4 - 4 * tid;
    uint4 sum = make_uint4(0, 0, 0, 0);
    const uint32_t addr = smem_u32(hist + bin0);
    for (int r = 0; r < ranks; ++r) {
      const uint4 v = ranks > 1 ? remote_u32x4(mapa_shared(addr, r)) : *reinterpret_cast<const uint4*>(hist + bin0);
      sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
    }
    uint32_t mine = sum.x + sum.y + sum.z + sum.w, upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const uint32_t x = __shfl_up_sync(0xffffffffu, upto, o); upto += lane >= o ? x : 0; }
    if (lane == 31) sm.warp_sum[0][warp] = upto;
    __syncthreads();
    for (int w = 0; w < warp; ++w) upto += sm.warp_sum[0][w];
    if (upto >= want && upto - mine < want) {                // the bin is one of this thread's
      uint32_t above = upto - mine;
      const uint32_t of[4] = {sum.w, sum.z, sum.y, sum.x};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (above < want && above + of[k] >= want) { sm.bin = (uint32_t)(bin0 + 3 - k); sm.above = above; sm.in_bin = of[k]; }
        above += of[k];
      }
    }
    __syncthreads();
    prefix = (prefix << bits) | sm.bin;
    want -= sm.above;
    least = prefix << shift; equal = want;                   // of the last pass: the order itself
    if (sm.in_bin == want) { least -= 1; equal = 0; break; } // the whole bin stays (never the lowest bin of all: more keys than stay)
    __syncthreads();
  }

  // numbers of what stays: a thread's keys lie one behind the other (an odd number of them: no two of a warp in one bank)
  const int seg = ((count + SEL_THREADS - 1) / SEL_THREADS) | 1, i0 = min(tid * seg, count), i1 = min(i0 + seg, count);
  uint32_t more = 0, same = 0;
  for (int i = i0; i < i1; ++i) { const uint32_t v = order_at(i); more += v > least; same += v == least; }
  uint32_t more_upto = more, same_upto = same;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t x = __shfl_up_sync(0xffffffffu, more_upto, o), y = __shfl_up_sync(0xffffffffu, same_upto, o);
    more_upto += lane >= o ? x : 0; same_upto += lane >= o ? y : 0;
  }
  __syncthreads();
  if (lane == 31) { sm.warp_sum[0][warp] = more_upto; sm.warp_sum[1][warp] = same_upto; }
  __syncthreads();
  for (int w = 0; w < warp; ++w) { more_upto += sm.warp_sum[0][w]; same_upto += sm.warp_sum[1][w]; }
  if (tid == SEL_THREADS - 1) { sm.taken[0] = more_upto; sm.taken[1] = same_upto; }
  uint32_t more_before = more_upto - more, same_before = same_upto - same;
  if (ranks > 1) {
    cluster_sync_all();
    for (int r = 0; r < rank; ++r) {
      more_before += remote_u32(mapa_shared(smem_u32(&sm.taken[0]), r));
      same_before += remote_u32(mapa_shared(smem_u32(&sm.taken[1]), r));
    }
  }
  for (int i = i0; i < i1; ++i) {
    const uint32_t v = order_at(i);
    const uint32_t to = rq.sinks + more_before + min(same_before, equal);
    if ((v > least || (v == least && same_before < equal)) && to < (uint32_t)t.a.budget) kept[to] = from + i;
    more_before += v > least; same_before += v == least;
  }
  // the first keys and the last ones
  const int recent = rq.length - rq.behind;
  for (int i = rank * SEL_THREADS + tid; i < rq.sinks; i += ranks * SEL_THREADS) kept[i] = i;
  for (int i = rank * SEL_THREADS + tid; i < recent; i += ranks * SEL_THREADS) kept[t.a.budget - recent + i] = rq.behind + i;
  if (ranks > 1) cluster_sync_all();                         // the others may still be reading this block's counts
}

// ---- moving together ---------------------------------------------------------------------------------------------------------

constexpr int MOVE_THREADS = 256, MOVE_ROWS = 4, MOVE_STAGES = 4;   // copies of a thread in a chunk, chunks on their way

// Copies of BYTES (16 or 4): thread i has piece i % pieces of row i / pieces, and of the rows a chunk's quarter further on.  row(place) is the address of
// a place's first byte of this block's columns, or null where its page is none of the pool's.
template <int BYTES, class RowOf>
__device__ __forceinline__ void move_rows(const EvictView& t, const int* kept, uint8_t* ring, int pieces, RowOf row) {
  const int tid = threadIdx.x, piece = tid % pieces, row_in = tid / pieces, rows = MOVE_THREADS / pieces, chunk = rows * MOVE_ROWS;
  const int chunks = (t.a.budget + chunk - 1) / chunk;
  uint8_t* const mine = ring + tid * BYTES;
  auto place_of = [&](int c, int k) { return c * chunk + k * rows + row_in; };
  int src[MOVE_ROWS];                                        // of the chunk that is fetched next
  auto ask = [&](int c) {
#pragma unroll
    for (int k = 0; k < MOVE_ROWS; ++k) { const int to = place_of(c, k); src[k] = to < t.a.budget ? kept[to] : -1; }
  };
  uint32_t moved = 0;                                        // which rows were fetched, of the chunks on their way
  auto fetch = [&](int c) {
    const int at = (c % MOVE_STAGES) * MOVE_ROWS;
    const uint8_t* from[MOVE_ROWS];
#pragma unroll
    for (int k = 0; k < MOVE_ROWS; ++k) from[k] = src[k] >= 0 && src[k] != place_of(c, k) ? row(src[k]) : nullptr;
#pragma unroll
    for (int k = 0; k < MOVE_ROWS; ++k) {
      moved = (moved & ~(1u << (at + k))) | (from[k] ? 1u << (at + k) : 0u);
      if (!from[k]) continue;
      const uint32_t to = smem_u32(mine + (at + k) * (MOVE_THREADS * BYTES));
      if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from[k] + piece * BYTES) : "memory");
      else asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to), "l"(from[k] + piece * BYTES) : "memory");
    }
  };
  ask(0);
  for (int c = 0; c < MOVE_STAGES - 1; ++c) {
    if (c < chunks) { fetch(c); ask(c + 1); }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  for (int c = 0; c < chunks; ++c) {
    const int ahead = c + MOVE_STAGES - 1;
    if (ahead < chunks) { fetch(ahead); ask(ahead + 1); }
    asm volatile("cp.async.commit_group;" ::: "memory");
    asm volatile("cp.async.wait_group %0;" ::"n"(MOVE_STAGES - 1) : "memory");
    __syncthreads();                                         // all of this chunk and of those before has been read
    const int at = (c % MOVE_STAGES) * MOVE_ROWS;
#pragma unroll
    for (int k = 0; k < MOVE_ROWS; ++k)
      if ((moved >> (at + k)) & 1) {
        const uint8_t* const from = mine + (at + k) * (MOVE_THREADS * BYTES);
        uint8_t* const to = row(place_of(c, k));
        if (to) {
          if (BYTES == 16) *reinterpret_cast<uint4*>(to + piece * BYTES) = *reinterpret_cast<const uint4*>(from);
          else *reinterpret_cast<uint32_t*>(to + piece * BYTES) = *reinterpret_cast<const uint32_t*>(from);
        }
      }
  }
}

__global__ void __launch_bounds__(MOVE_THREADS) evict_move_kernel(const EvictView t) {
  extern __shared__ __align__(16) uint8_t smem_bytes[];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int h = blockIdx.y, b = blockIdx.z, stream = blockIdx.x;
  const int* const kept = t.a.kept_out + ((long long)b * t.c.num_kv_heads + h) * t.a.budget;
  const bool weights = stream == 2 * t.slices;
  // the one reader of this request's length in this launch, so that lengths_out may be lengths
  if (weights && h == 0 && threadIdx.x == 0) t.a.lengths_out[b] = min(evict_request(t, b).length, t.a.budget);
  if (kept[t.a.budget - 1] < t.a.budget) return;             // at most `budget` keys: all where they are
  const int* const table = t.c.block_table + (long long)b * t.c.table_stride;
  auto page_of = [&](int place, int* slot) {
    const int col = page_column(t, place), page = table[col];
    *slot = place - col * t.c.page_size;
    if ((unsigned)page < (unsigned)t.c.num_pages) return page;
    cache_report(t.c, CACHE_BAD_PAGE);
    return -1;
  };
  if (weights) {
    move_rows<4>(t, kept, smem_bytes, 1, [&](int place) -> uint8_t* {
      int slot;
      const int page = page_of(place, &slot);
      return page < 0 ? nullptr : reinterpret_cast<uint8_t*>(t.a.weights + ((long long)page * t.c.num_kv_heads + h) * t.c.page_size + slot);
    });
  } else {
    const int which = stream / t.slices, row_bytes = t.c.key_size * 2, bytes = row_bytes / t.slices, column = (stream % t.slices) * bytes;
    move_rows<16>(t, kept, smem_bytes, bytes / 16, [&](int place) -> uint8_t* {
      int slot;
      const int page = page_of(place, &slot);
      return page < 0 ? nullptr : reinterpret_cast<uint8_t*>(t.c.pages) + (cache_row0(t.c, page, which, h) * 2 + (long long)slot * row_bytes + column);
    });
  }
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
  if (t.a.max_keys < 0) return bad("negative size");
  if (t.c.batch == 0) return PHX_OK;
  if (!t.a.weights || !t.a.lengths_out || !t.a.kept_out) return bad("weights, lengths_out and kept_out are required");
  const long long columns = (long long)t.c.table_cols * t.c.page_size;
  if (t.a.max_keys > columns) t.a.max_keys = columns;
  const int e = t.c.page_size / 16;
  t.page_magic = ((1ull << 36) + e - 1) / e;
  DeviceScope scope(device);
  if (!scope.ok()) { set_global_error("phx_evict_device: cudaSetDevice failed"); return PHX_E_CUDA; }
  cudaStream_t st = (cudaStream_t)stream;
  const long long heads = (long long)t.c.batch * t.c.num_kv_heads;

  // Blocks of a cluster: as long as the heads' clusters fit the device twice over and a block keeps 1024 weights
  int ranks = 1;
  while (ranks < 8 && heads * ranks * 2 <= 2ll * device_sms() && t.a.max_keys / ranks > 1024) ranks *= 2;
  constexpr int MOST_HELD = 48 * 1024;                        // weights: 192 KB beside the histograms; longer stretches are read from memory at each pass
  const long long per = (t.a.max_keys + ranks - 1) / ranks;
  t.held = (int)(per < MOST_HELD ? per : MOST_HELD);
  // Columns of a head's rows are shared between blocks until the device has two blocks an SM; a block copies 64 bytes of a row at least
  t.slices = 1;
  while (heads * 2 * t.slices < 2ll * device_sms() && t.c.key_size * 2 / (2 * t.slices) >= 64) t.slices *= 2;
  const int select_smem = (int)sizeof(SelectSmem) + t.held * 4, move_smem = MOVE_STAGES * MOVE_ROWS * MOVE_THREADS * 16;
  static SmemLimit select_limit, move_limit;
  std::string err;
  auto launch = [&]() -> phx_status {
    PHX_CUDA_TRY(select_limit.raise(evict_select_kernel, (int)sizeof(SelectSmem) + MOST_HELD * 4), err);
    PHX_CUDA_TRY(move_limit.raise(evict_move_kernel, move_smem), err);
    cudaLaunchConfig_t lc;
    memset(&lc, 0, sizeof(lc));
    lc.gridDim = dim3(ranks, t.c.num_kv_heads, t.c.batch); lc.blockDim = dim3(SEL_THREADS); lc.dynamicSmemBytes = select_smem; lc.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ranks; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    lc.attrs = at; lc.numAttrs = 1;
    PHX_CUDA_TRY(cudaLaunchKernelEx(&lc, evict_select_kernel, t), err);
    PHX_CUDA_TRY(launch_programmatic(evict_move_kernel, dim3(2 * t.slices + 1, t.c.num_kv_heads, t.c.batch), dim3(MOVE_THREADS), move_smem, st, t), err);
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
