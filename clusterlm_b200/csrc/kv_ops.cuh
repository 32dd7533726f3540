// kv_ops.cuh — the paged KV cache as operators over caller-owned memory: page pools, page tables, positions.
//
// A page holds kPageTokens (64) positions of every kv head of one layer: K [n_kv][64][hd] and V^T [n_kv][hd][64],
// 16-byte chunks permuted as in llama.cuh (kv_k_chunk, kv_v_chunk), the layout of the engines' own caches.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>
#include <vector>

#include "common.cuh"
#include "llama.cuh"

namespace clm {

constexpr int kKvMaxSeqs = 512;     // sequences of one call
constexpr int kKvMaxGroups = 64;    // groups of sequences that share leading pages
constexpr int kKvMaxWindow = 256;   // rows of one sequence in one attention call (the engines' widest window)
constexpr int kKvMaxMapped = 16;    // sequences of a call that names table rows by slot (an engine's sessions)

// The sequences of a call: row b of the page tables and its committed position.  Tables and positions are read on the
// device, so a captured graph replays with their current contents.
struct KvSeqs {
  const int32_t* tables = nullptr;
  long long table_stride = 0;  // entries between the tables of consecutive slots
  const char* pos = nullptr;   // long long at pos + slot * pos_stride
  long long pos_stride = sizeof(long long);
  int n = 0;
  int max_pages = 0;   // entries of a table
  int pool_pages = 0;  // pages of the pool: an entry outside [0, pool_pages) is no page
  int mapped = 0;      // 1: sequence b is slot[b], else slot b
  uint16_t slot[kKvMaxMapped] = {};
  __device__ __forceinline__ int at(int b) const { return mapped ? slot[b] : b; }
  // (held at 2^62, far behind every table, so that sums with a window's rows do not wrap)
  __device__ __forceinline__ long long base(int b) const {
    return min(*reinterpret_cast<const long long*>(pos + (long long)at(b) * pos_stride), 1ll << 62);
  }
  __device__ __forceinline__ const int32_t* table(int b) const { return tables + (long long)at(b) * table_stride; }
};

// Sequences [start[g], start[g + 1]) share the first pages[g] table entries.
struct KvGroups {
  int n = 0;
  uint16_t start[kKvMaxGroups + 1] = {};
  uint32_t pages[kKvMaxGroups] = {};
};

struct KvAttnArgs {
  KvSeqs seqs;
  KvGroups groups;
  const void* k = nullptr;  // this layer's pools
  const void* v = nullptr;
  const void* q = nullptr;  // [n][positions][nh][hd], consecutive rows ld_q elements apart
  long long ld_q = 0;
  void* out = nullptr;  // [n][positions][nh][hd]
  const int32_t* parent = nullptr;
  int positions = 0, nh = 0, nkv = 0, hd = 0;
  int type = CLM_DTYPE_F16;      // of q and the pools
  int out_type = CLM_DTYPE_F16;  // the same, or f32 (engines)
  float scale = 0.0f;
  void* work = nullptr;
  size_t work_bytes = 0;
  int sm_count = 148;
  uint32_t polls = kAttentionPolls;  // a wait inside gives up after so many polls: rows of NaN, and
  int* err = nullptr;                // (device) kErrWaitTimeout here
};
// Workspace bytes of launch_kv_attention (an upper bound over the device-side lengths).
size_t kv_attention_work(int n, int positions, int nh, int nkv, int hd, const KvGroups& groups, int sm_count);
int launch_kv_attention(const KvAttnArgs& a, cudaStream_t st);

// Page copies: pool page src[i] -> dst[i] in every layer of K and V; with tables, entries naming src[i] then name
// dst[i].  At most kKvCopyMax pairs a launch.
constexpr int kKvCopyMax = 256;
struct KvCopyJob {
  int n = 0;
  int32_t src[kKvCopyMax], dst[kKvCopyMax];
};
int launch_kv_copy(void* k, void* v, uint32_t layers, uint64_t layer_bytes, uint64_t page_bytes, const KvCopyJob& job,
                   int32_t* tables, uint64_t table_entries, int sm_count, cudaStream_t st);

// Host ledger of a pool's pages: reference counts and the free pages (lowest page first).
class PageLedger {
 public:
  explicit PageLedger(uint32_t pages) : refs_(pages, 0), free_(pages) {}
  uint32_t pages() const { return (uint32_t)refs_.size(); }
  uint32_t free_count() const { return free_; }
  uint32_t refs(uint32_t id) const { return refs_[id]; }
  bool valid(int32_t id) const { return id >= 0 && (size_t)id < refs_.size(); }
  // n free pages (one reference each), lowest first; false (and nothing taken) when fewer are free
  bool alloc(uint32_t n, int32_t* out);
  void retain(int32_t id) { ++refs_[id]; }
  void release(int32_t id);
  void restore(int32_t id) {  // undoes a release
    if (refs_[id]++ == 0) --free_;
  }
  // Moves that pack the live pages into [0, live): pairs (src, dst), references moved along.
  void compact(std::vector<int32_t>& src, std::vector<int32_t>& dst);

 private:
  std::vector<uint32_t> refs_;
  uint32_t free_;
  uint32_t first_ = 0;  // no free page below this one
};

int check_kv_pool(const clm_b200_kv_pool* p);
int check_kv_seqs(const clm_b200_kv_seqs* s);
uint64_t kv_page_bytes(const clm_b200_kv_pool* p);  // of one layer's K, or V
KvSeqs make_kv_seqs(const clm_b200_kv_pool* pool, const clm_b200_kv_seqs* s, uint32_t n);

inline size_t dtype_size(int t) { return t == CLM_DTYPE_F32 ? 4 : 2; }

// Makes a context's device current for a call and the caller's own device again at its end.
class DeviceScope {
 public:
  explicit DeviceScope(int device) {
    if (cudaGetDevice(&before_) != cudaSuccess) before_ = -1;
    if (before_ != device) {
      rc_ = cudaSetDevice(device);
      changed_ = rc_ == cudaSuccess;
    }
  }
  ~DeviceScope() {
    if (changed_ && before_ >= 0) cudaSetDevice(before_);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
  cudaError_t status() const { return rc_; }

 private:
  int before_ = -1;
  bool changed_ = false;
  cudaError_t rc_ = cudaSuccess;
};

#define CLM_SCOPE(ctx)                                                                  \
  CLM_CHECK((ctx) != nullptr, CLM_INVALID_ARGUMENT, "null context");                    \
  ::clm::DeviceScope clm_scope_((ctx)->device);                                         \
  if (clm_scope_.status() != cudaSuccess) return ::clm::cuda_fail(clm_scope_.status(), "cudaSetDevice")

// ---- element conversions of the operators' types
template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// two values, the first in the low half
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

}  // namespace clm
