// What the operators on a paged cache share: the checks of a phx_cache_batch on the host, its lookups on the device.
#pragma once

#include "common.cuh"

namespace phx {

constexpr int CACHE_BAD_PAGE = 1, CACHE_BAD_POSITION = 2, CACHE_BAD_OFFSETS = 4;   // bits of status_dev[2]

__device__ __forceinline__ void cache_report(const phx_cache_batch& c, int bit) { atomicOr(c.status_dev + 2, bit); }

// new tokens and older keys of request b; offsets that leave the token rows make it an empty request
struct CacheRequest { int row0, tokens, cached; bool ok; };
__device__ __forceinline__ CacheRequest cache_request(const phx_cache_batch& c, int b) {
  const int r0 = c.q_start[b], r1 = c.q_start[b + 1], len = c.lengths[b];
  const bool ok = r0 >= 0 && r1 >= r0 && r1 <= c.num_tokens && len >= 0;
  CacheRequest q;
  q.ok = ok;
  q.row0 = ok ? r0 : 0; q.tokens = ok ? r1 - r0 : 0; q.cached = ok ? len : 0;
  return q;
}
// keys that the request's row of the table has columns for
__device__ __forceinline__ long long cache_columns(const phx_cache_batch& c) { return (long long)c.table_cols * c.page_size; }
// first element of head `h`'s rows in a page: which = 0 keys, 1 values
__device__ __forceinline__ long long cache_row0(const phx_cache_batch& c, long long page, int which, int h) {
  return ((page * 2 + which) * c.num_kv_heads + h) * (long long)c.page_size * c.key_size;
}

// "" or what is wrong with the batch
inline const char* cache_check(const phx_cache_batch* c) {
  if (!c) return "null argument";
  if (c->batch < 0 || c->num_tokens < 0 || c->num_pages < 0 || c->table_cols < 0) return "negative size";
  if (c->key_size != 32 && c->key_size != 64 && c->key_size != 128) return "key_size must be 32, 64 or 128";
  if (c->num_kv_heads < 1 || c->num_kv_heads > 1024) return "num_kv_heads must be 1 to 1024";
  if (c->page_size < 16 || c->page_size % 16 != 0 || c->page_size > 4096) return "page_size must be a multiple of 16, at most 4096";
  if (!c->status_dev) return "status_dev is required";
  if (c->batch == 0 || c->num_tokens == 0) return "";
  if (!c->q_start || !c->lengths) return "q_start and lengths are required";
  if (c->table_cols > 0 && (!c->block_table || c->table_stride < c->table_cols)) return "block_table is required, its rows at least table_cols apart";
  if (c->num_pages > 0 && (!c->pages || (reinterpret_cast<uintptr_t>(c->pages) & 15) != 0)) return "pages must be a 16-byte aligned pool";
  if ((long long)c->table_cols * c->page_size > 2147483647ll - 4096) return "a request's keys must fit 31 bits";
  if (c->num_pages > 2147483647ll / (2ll * c->num_kv_heads * c->page_size)) return "the pool's rows (pages x 2 x heads x page_size) must fit 31 bits";
  return "";
}
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// `e`; a failure is the entry point's answer, so it is taken back as the runtime's last error, which the next launch would report as its own
inline cudaError_t taken_back(cudaError_t e) {
  if (e != cudaSuccess) (void)cudaGetLastError();
  return e;
}

// makes `device` current for the calls of one entry point and puts the caller's back
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    ok_ = taken_back(cudaGetDevice(&before_)) == cudaSuccess && (before_ == device || taken_back(cudaSetDevice(device)) == cudaSuccess);
    changed_ = ok_ && before_ != device;
  }
  ~DeviceScope() { if (changed_) cudaSetDevice(before_); }
  bool ok() const { return ok_; }
 private:
  int before_ = 0;
  bool ok_ = false, changed_ = false;
};

}  // namespace phx
