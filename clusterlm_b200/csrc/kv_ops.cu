// kv_ops.cu — operators on a paged KV cache: rows in (with rotary positions), forks, page copies, the page ledger.
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "kv_ops.cuh"
#include "pdl.cuh"

namespace clm {

// ---------------------------------------------------------------------------------------------------
// kv_append: rotate q and k, write k and v into their pages
//
// A rotated pair (x, y) of frequency f at position P becomes s (x cos(P f) - y sin(P f), x sin(P f) + y cos(P f)).
// P f is formed and reduced modulo 2 pi in double (at P = 10^6 an f32 angle is off by 0.03 rad); the reduced angle's
// sine and cosine are f32.  Products are f32 and round once to the cache's type.
//
// One CTA per (sequence, quarter page that its rows touch, range of kv heads): the rows' angles are evaluated once into
// shared memory and serve all its heads; the value rows are transposed through shared memory, because a V page keeps a
// dimension's 64 positions together: two threads write a quarter's 32 bytes.
//
// Bound by memory.  4,096 rows of 64 + 8 + 8 heads of 128, f32 to bf16 (252 MB): 47 us, 5.4 TB/s; with 256 threads a
// CTA 56 us, with 64 58 us; with a CTA per (page, kv head), whose angles are evaluated once per kv head, 65 us.  16
// sequences of 4 rows (1.6 MB): 6 us, a launch and three dependent reads.
// ---------------------------------------------------------------------------------------------------
namespace {

constexpr int kAppendThreads = 128;
constexpr int kAppendRows = 16;   // positions of a CTA: a quarter page
constexpr int kAppendHeads = 8;   // kv heads of a CTA at most

struct AppendArgs {
  KvSeqs seqs;
  const void *q, *k, *v;
  long long ld_q, ld_k, ld_v;
  void *q_out, *kpool, *vpool;
  const double* freq;
  const int32_t* parent;
  float scale;
  int positions, nh, nkv, hd, rot, interleaved, blocks, heads;  // CTAs of a sequence; kv heads of a CTA
  int vec_q, vec_k, vec_v;  // rows start 16-byte aligned: vector loads
};

template <typename S>
__device__ __forceinline__ void load8(const S* p, bool vec, float (&x)[8]) {
  if (vec) {
    if constexpr (sizeof(S) == 4) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const S* e = reinterpret_cast<const S*>(&w[i]);
        x[2 * i] = to_f32(e[0]);
        x[2 * i + 1] = to_f32(e[1]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = to_f32(p[i]);
  }
}

template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
}

// Elements [d0, d0 + 8) of a head's row `p` after the rotation; cs[j] = (cos, sin) of the row's pair j.  (Rotations
// whose halves are not whole chunks; rotate_rows has the others.)
template <typename S>
__device__ __forceinline__ void rotate8(const S* p, int d0, const AppendArgs& a, bool vec, const float2* cs,
                                        float (&o)[8]) {
  float x[8];
  load8(p + d0, vec, x);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int d = d0 + i, half = a.rot / 2;
    if (d >= a.rot) {
      o[i] = x[i];
    } else if (a.interleaved) {
      const float2 c = cs[d / 2];
      o[i] = i % 2 == 0 ? x[i] * c.x - x[i + 1 & 7] * c.y : x[i - 1 & 7] * c.y + x[i] * c.x;
    } else if (d < half) {
      const float2 c = cs[d];
      o[i] = x[i] * c.x - to_f32(p[d + half]) * c.y;
    } else {
      const float2 c = cs[d - half];
      o[i] = to_f32(p[d - half]) * c.y + x[i] * c.x;
    }
  }
}

// Runs over the (row, head, unit)s of a page's rows, a thread every kAppendThreads-th: carried along, not divided for.
struct RowWalk {
  int r, h, u;
  int heads, units, dr, dh, du;
  __device__ __forceinline__ RowWalk(int n_heads, int n_units) : heads(n_heads), units(n_units) {
    const int per = heads * units;
    r = threadIdx.x / per, dr = kAppendThreads / per;
    const int x = threadIdx.x % per, y = kAppendThreads % per;
    h = x / units, dh = y / units;
    u = x % units, du = y % units;
  }
  __device__ __forceinline__ void next() {
    u += du, h += dh, r += dr;
    if (u >= units) u -= units, ++h;
    if (h >= heads) h -= heads, ++r;
  }
};

// Rotates the heads' rows [0, nr) of `src` and gives their chunks to store(row, head, first element, values).  With
// halves of whole chunks a unit is a chunk of the first half and its partner: each element is read once, and two
// units' loads are in flight.
template <typename S, typename F>
__device__ __forceinline__ void rotate_rows(const S* src, long long ld, int heads, int nr, const AppendArgs& a, bool vec,
                                            const float2* cs, F&& store) {
  const int half = a.rot / 2, hd = a.hd;
  if (a.interleaved ? a.rot % 8 == 0 : half % 8 == 0) {
    const int pairs = a.interleaved ? a.rot / 8 : half / 8;  // units that rotate; the rest are chunks that stay
    RowWalk w(heads, pairs + (hd - a.rot) / 8);
    while (w.r < nr) {
      float x[2][8], y[2][8];
      int r[2], h[2], d[2];
      bool turn[2], two[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        r[q] = w.r, h[q] = w.h;
        turn[q] = w.u < pairs;
        two[q] = turn[q] && !a.interleaved;
        d[q] = turn[q] ? 8 * w.u : a.rot + 8 * (w.u - pairs);
        if (r[q] < nr) {
          const S* p = src + (long long)r[q] * ld + h[q] * hd + d[q];
          load8(p, vec, x[q]);
          if (two[q]) load8(p + half, vec, y[q]);
        }
        w.next();
      }
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (r[q] >= nr) continue;
        float o[8];
        if (two[q]) {
          const float2* c8 = cs + r[q] * half + d[q];
          float o2[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float2 c = c8[i];
            o[i] = x[q][i] * c.x - y[q][i] * c.y;
            o2[i] = x[q][i] * c.y + y[q][i] * c.x;
          }
          store(r[q], h[q], d[q] + half, o2);
        } else if (turn[q]) {
          const float2* c4 = cs + r[q] * half + d[q] / 2;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float2 c = c4[i];
            o[2 * i] = x[q][2 * i] * c.x - x[q][2 * i + 1] * c.y;
            o[2 * i + 1] = x[q][2 * i] * c.y + x[q][2 * i + 1] * c.x;
          }
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) o[i] = x[q][i];
        }
        store(r[q], h[q], d[q], o);
      }
    }
    return;
  }
  for (RowWalk w(heads, hd / 8); w.r < nr; w.next()) {
    float o[8];
    rotate8(src + (long long)w.r * ld + w.h * hd, 8 * w.u, a, vec, cs + w.r * half, o);
    store(w.r, w.h, 8 * w.u, o);
  }
}

template <typename S, typename T>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const __grid_constant__ AppendArgs a) {
  extern __shared__ __align__(16) uint8_t ap_smem[];
  __shared__ int s_depth[kAppendRows];
  griddep_wait();
  griddep_launch();
  const int b = blockIdx.x / a.blocks, c = blockIdx.x % a.blocks, kv0 = blockIdx.y * a.heads;
  const int kvn = min(a.heads, a.nkv - kv0), group = a.nh / a.nkv, hd = a.hd, half = a.rot / 2;
  float2* cs = reinterpret_cast<float2*>(ap_smem);  // [16][half]
  const int vld = hd + 2;                           // padded row of the value tiles, elements
  T* vt = reinterpret_cast<T*>(ap_smem + (size_t)kAppendRows * half * sizeof(float2));  // [heads][16][vld]
  const long long base = a.seqs.base(b);
  const S* q = static_cast<const S*>(a.q);
  T* q_out = static_cast<T*>(a.q_out);
  const int g0 = b * a.positions;  // the sequence's first row
  if (base < 0) {                  // an idle sequence: nothing enters the cache, its query rows become zero
    const int r0 = c * kAppendRows, nr = min(kAppendRows, a.positions - r0), per = kvn * group * hd / 8;
    if (q != nullptr)
      for (int i = threadIdx.x; i < nr * per; i += kAppendThreads)
        *reinterpret_cast<uint4*>(q_out + ((size_t)(g0 + r0 + i / per) * a.nh + kv0 * group) * hd + 8 * (i % per)) =
            make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  const long long block = base / kAppendRows + c, pg = block / (kPageTokens / kAppendRows);
  const long long lo = max(base, block * kAppendRows), hi = min(base + a.positions, (block + 1) * kAppendRows);
  const int r0 = (int)(lo - base), nr = (int)(hi - lo);  // rows r0 .. r0 + nr - 1 of the window lie in this block
  if (nr <= 0) return;
  const int at0 = (int)(block % (kPageTokens / kAppendRows)) * kAppendRows;  // the block's first position in the page
  const int p0 = (int)(lo % kAppendRows);                                    // the first row's place in the block
  int32_t page = pg < a.seqs.max_pages ? a.seqs.table(b)[pg] : -1;
  if (page >= a.seqs.pool_pages) page = -1;  // no page: the rows are rotated but not kept
  for (int r = threadIdx.x; r < nr; r += kAppendThreads) {
    int d = r0 + r;
    if (a.parent != nullptr) {  // depth of tree node r0 + r (an entry that is not an earlier node ends the walk)
      int at = r0 + r;
      for (d = 0;; ++d) {
        const int up = a.parent[at];
        if (up < 0 || up >= at) break;
        at = up;
      }
    }
    s_depth[r] = d;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < nr * half; i += kAppendThreads) {
    const int r = i / half, j = i % half;
    const double angle = (double)(base + s_depth[r]) * a.freq[j];
    const double turns = rint(angle * 0.15915494309189535);  // 1 / (2 pi)
    double red = fma(-turns, 6.283185307179586, angle);
    red = fma(-turns, 2.4492935982947064e-16, red);  // the rest of 2 pi
    float sn, cn;
    sincosf((float)red, &sn, &cn);
    cs[i] = make_float2(cn * a.scale, sn * a.scale);
  }
  // the value tiles, rows at their place in the block (with the angles: one barrier for both)
  if (page >= 0) {
    const S* v = static_cast<const S*>(a.v) + (long long)(g0 + r0) * a.ld_v + kv0 * hd;
#pragma unroll 2
    for (RowWalk w(kvn, hd / 8); w.r < nr; w.next()) {
      float x[8];
      load8(v + (long long)w.r * a.ld_v + w.h * hd + 8 * w.u, a.vec_v, x);
      uint32_t* t = reinterpret_cast<uint32_t*>(vt + (size_t)(w.h * kAppendRows + p0 + w.r) * vld + 8 * w.u);
#pragma unroll
      for (int k = 0; k < 4; ++k) t[k] = pack2<T>(x[2 * k], x[2 * k + 1]);
    }
  }
  __syncthreads();
  if (q != nullptr)
    rotate_rows(q + (long long)(g0 + r0) * a.ld_q + kv0 * group * hd, a.ld_q, kvn * group, nr, a, a.vec_q, cs,
                [&](int r, int h, int d, const float(&o)[8]) {
                  *reinterpret_cast<uint4*>(q_out + ((size_t)(g0 + r0 + r) * a.nh + kv0 * group + h) * hd + d) = pack8<T>(o);
                });
  if (page < 0) return;
  const size_t at = ((size_t)page * a.nkv + kv0) * kPageTokens * hd;
  T* kp = static_cast<T*>(a.kpool) + at;
  T* vp = static_cast<T*>(a.vpool) + at;
  rotate_rows(static_cast<const S*>(a.k) + (long long)(g0 + r0) * a.ld_k + kv0 * hd, a.ld_k, kvn, nr, a, a.vec_k, cs,
              [&](int r, int h, int d, const float(&o)[8]) {
                const int pos = at0 + p0 + r;
                *reinterpret_cast<uint4*>(kp + (size_t)(h * kPageTokens + pos) * hd + 8 * kv_k_chunk(d / 8, pos)) = pack8<T>(o);
              });
  // chunks of 8 positions of a dimension, two a block
  for (int i = threadIdx.x; i < 2 * kvn * hd; i += kAppendThreads) {
    const int pc = i % 2, d = i / 2 % hd, h = i / 2 / hd;
    const T* from = vt + (size_t)(h * kAppendRows + 8 * pc) * vld + d;
    T* dst = vp + (size_t)(h * hd + d) * kPageTokens + 8 * kv_v_chunk(at0 / 8 + pc, d);
    if (8 * pc >= p0 && 8 * pc + 8 <= p0 + nr) {
      T e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = from[(size_t)j * vld];
      uint4 w;
      memcpy(&w, e, 16);
      *reinterpret_cast<uint4*>(dst) = w;
    } else {  // a chunk that other rows share: the other positions stay as they are
      for (int j = 0; j < 8; ++j)
        if (8 * pc + j >= p0 && 8 * pc + j < p0 + nr) dst[j] = from[(size_t)j * vld];
    }
  }
}

// ---------------------------------------------------------------------------------------------------
// page copies and forks: every layer's K and V page of each pair, 8 KB units spread over the grid, four units
// (eight 16-byte loads a thread) in flight per CTA.  Bound by memory: 384 pages of 10 layers (2 GB read and written)
// 304 us, 6.6 TB/s, with up to 64 CTAs per SM one after the other (8 persistent ones 344 us, 32 310 us); eight forks
// of one parent (67 MB written) 15 us, its page read from the cache seven times (with streaming loads 21 us).
// ---------------------------------------------------------------------------------------------------
constexpr int kCopyThreads = 256;
constexpr int kCopyUnit = 8192;   // bytes: a page is a whole number of them (64 positions x 64 dims x 2 bytes)
constexpr int kCopyBatch = 4;

struct ForkJob {
  int n = 0;
  uint16_t parent[kKvCopyMax], child[kKvCopyMax];
  int32_t page[kKvCopyMax];
};

struct SlabArgs {
  uint8_t *k, *v;
  uint64_t layer_bytes, page_bytes;
  uint32_t layers;
};

__device__ __forceinline__ void copy_pages(const SlabArgs& s, const int32_t* src, const int32_t* dst, int n) {
  const uint32_t upp = (uint32_t)(s.page_bytes / kCopyUnit);  // units per page of one layer of K or V
  const uint64_t per = (uint64_t)upp * 2 * s.layers, total = per * n;
  for (uint64_t u0 = (uint64_t)blockIdx.x * kCopyBatch; u0 < total; u0 += (uint64_t)gridDim.x * kCopyBatch) {
    uint4 x[2 * kCopyBatch];
    uint4* to[kCopyBatch];
#pragma unroll
    for (int j = 0; j < kCopyBatch; ++j) {
      const uint64_t u = u0 + j;
      to[j] = nullptr;
      if (u >= total) continue;
      const int job = (int)(u / per);
      const uint32_t rest = (uint32_t)(u % per), slab = rest / upp, part = rest % upp;
      if (src[job] < 0) continue;
      uint8_t* base = (slab & 1 ? s.v : s.k) + (uint64_t)(slab >> 1) * s.layer_bytes + (uint64_t)part * kCopyUnit;
      const uint4* from = reinterpret_cast<const uint4*>(base + (uint64_t)src[job] * s.page_bytes);
      to[j] = reinterpret_cast<uint4*>(base + (uint64_t)dst[job] * s.page_bytes);
      x[2 * j] = __ldg(from + threadIdx.x);
      x[2 * j + 1] = __ldg(from + kCopyThreads + threadIdx.x);
    }
#pragma unroll
    for (int j = 0; j < kCopyBatch; ++j)
      if (to[j] != nullptr) {
        to[j][threadIdx.x] = x[2 * j];
        to[j][kCopyThreads + threadIdx.x] = x[2 * j + 1];
      }
  }
}

__global__ void __launch_bounds__(kCopyThreads) kv_copy_kernel(SlabArgs s, const __grid_constant__ KvCopyJob job,
                                                               int32_t* __restrict__ tables, uint64_t entries) {
  __shared__ int32_t s_src[kKvCopyMax], s_dst[kKvCopyMax];
  for (int i = threadIdx.x; i < job.n; i += kCopyThreads) {
    s_src[i] = job.src[i];
    s_dst[i] = job.dst[i];
  }
  __syncthreads();
  griddep_wait();
  griddep_launch();
  // the tables' entries follow the pages (s_src ascends)
  for (uint64_t i = blockIdx.x * (uint64_t)kCopyThreads + threadIdx.x; i < entries;
       i += (uint64_t)gridDim.x * kCopyThreads) {
    const int32_t t = tables[i];
    int lo = 0, hi = job.n;
    while (lo < hi) {
      const int mid = (lo + hi) / 2;
      if (s_src[mid] < t)
        lo = mid + 1;
      else
        hi = mid;
    }
    if (lo < job.n && s_src[lo] == t) tables[i] = s_dst[lo];
  }
  copy_pages(s, s_src, s_dst, job.n);
}

__global__ void __launch_bounds__(kCopyThreads) kv_fork_kernel(SlabArgs s, const __grid_constant__ ForkJob job,
                                                               int32_t* __restrict__ tables, int max_pages,
                                                               int pool_pages, long long* __restrict__ pos) {
  __shared__ int32_t s_src[kKvCopyMax], s_dst[kKvCopyMax];
  griddep_wait();
  griddep_launch();
  for (int i = threadIdx.x; i < job.n; i += kCopyThreads) {
    const long long p = pos[job.parent[i]], full = p / kPageTokens;
    int32_t src = -1;
    if (p >= 0 && p % kPageTokens != 0 && full < max_pages) {
      src = tables[(uint64_t)job.parent[i] * max_pages + full];
      if (src >= pool_pages) src = -1;
    }
    s_src[i] = src;
    s_dst[i] = job.page[i];
  }
  __syncthreads();
  // CTA i writes child i's table and position (no child is a parent of the same call)
  for (int i = blockIdx.x; i < job.n; i += gridDim.x) {
    const long long p = pos[job.parent[i]];
    const int32_t* from = tables + (uint64_t)job.parent[i] * max_pages;
    int32_t* to = tables + (uint64_t)job.child[i] * max_pages;
    if (p >= 0) {
      const long long full = p / kPageTokens < max_pages ? p / kPageTokens : max_pages;
      for (int e = threadIdx.x; e < full; e += kCopyThreads) to[e] = from[e];
      if (threadIdx.x == 0 && full < max_pages) to[full] = job.page[i];
    }
    if (threadIdx.x == 0) pos[job.child[i]] = p;
  }
  copy_pages(s, s_src, s_dst, job.n);
}

unsigned copy_grid(uint64_t page_bytes, uint32_t layers, int n, int sm_count) {
  const uint64_t units = (uint64_t)n * layers * 2 * (page_bytes / kCopyUnit);
  const uint64_t ctas = ceil_div(units, kCopyBatch);
  return (unsigned)std::max<uint64_t>(1, std::min<uint64_t>(ctas, (uint64_t)sm_count * 64));
}

}  // namespace

int launch_kv_copy(void* k, void* v, uint32_t layers, uint64_t layer_bytes, uint64_t page_bytes, const KvCopyJob& job,
                   int32_t* tables, uint64_t table_entries, int sm_count, cudaStream_t st) {
  if (job.n == 0) return CLM_OK;
  const SlabArgs s{static_cast<uint8_t*>(k), static_cast<uint8_t*>(v), layer_bytes, page_bytes, layers};
  return launch_pdl(kv_copy_kernel, dim3(copy_grid(page_bytes, layers, job.n, sm_count)), dim3(kCopyThreads), 0, st, s,
                    job, tables, tables ? table_entries : 0ull);
}

// ---------------------------------------------------------------------------------------------------
// page ledger (host)
// ---------------------------------------------------------------------------------------------------
bool PageLedger::alloc(uint32_t n, int32_t* out) {
  if (n > free_) return false;
  for (uint32_t i = 0; i < n; ++i) {
    while (refs_[first_] != 0) ++first_;
    refs_[first_] = 1;
    out[i] = (int32_t)first_;
  }
  free_ -= n;
  return true;
}

void PageLedger::release(int32_t id) {
  if (--refs_[id] == 0) {
    ++free_;
    first_ = std::min(first_, (uint32_t)id);
  }
}

void PageLedger::compact(std::vector<int32_t>& src, std::vector<int32_t>& dst) {
  const uint32_t live = pages() - free_;
  uint32_t to = 0;
  for (uint32_t from = live; from < pages(); ++from) {
    if (refs_[from] == 0) continue;
    while (refs_[to] != 0) ++to;  // below `live` there is a free page for every live page at or above it
    src.push_back((int32_t)from);
    dst.push_back((int32_t)to);
    refs_[to] = refs_[from];
    refs_[from] = 0;
  }
  first_ = live;
}

// ---------------------------------------------------------------------------------------------------
// argument checks that the cache's operators share
// ---------------------------------------------------------------------------------------------------
int check_kv_pool(const clm_b200_kv_pool* p) {
  CLM_CHECK(p != nullptr && p->k != nullptr && p->v != nullptr, CLM_INVALID_ARGUMENT, "null pool");
  CLM_CHECK(p->layers >= 1 && p->pages >= 1 && p->n_kv_heads >= 1, CLM_INVALID_ARGUMENT, "empty pool");
  CLM_CHECK(p->pages <= 0x7fffffffu, CLM_OUT_OF_RANGE, "a pool has at most 2^31 - 1 pages");
  CLM_CHECK(p->dtype == CLM_DTYPE_F16 || p->dtype == CLM_DTYPE_BF16, CLM_UNIMPLEMENTED, "a pool holds f16 or bf16");
  CLM_CHECK(p->head_dim == 64 || p->head_dim == 128, CLM_UNIMPLEMENTED, "head_dim 64 or 128");
  CLM_CHECK(p->n_kv_heads <= 65535, CLM_OUT_OF_RANGE, "at most 65535 kv heads");
  CLM_CHECK(((reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v)) & 15) == 0, CLM_INVALID_ARGUMENT,
            "pools must be 16-byte aligned");
  return CLM_OK;
}

uint64_t kv_page_bytes(const clm_b200_kv_pool* p) { return (uint64_t)p->n_kv_heads * kPageTokens * p->head_dim * 2; }

int check_kv_seqs(const clm_b200_kv_seqs* s) {
  CLM_CHECK(s != nullptr && s->d_tables != nullptr && s->d_pos != nullptr, CLM_INVALID_ARGUMENT, "null sequences");
  CLM_CHECK(s->rows >= 1 && s->max_pages >= 1 && s->max_pages <= (1u << 25), CLM_INVALID_ARGUMENT,
            "empty page tables, or more than 2^25 pages a sequence");
  return CLM_OK;
}

KvSeqs make_kv_seqs(const clm_b200_kv_pool* pool, const clm_b200_kv_seqs* s, uint32_t n) {
  KvSeqs r;
  r.tables = s->d_tables;
  r.table_stride = s->max_pages;
  r.pos = reinterpret_cast<const char*>(s->d_pos);
  r.n = (int)n;
  r.max_pages = (int)s->max_pages;
  r.pool_pages = (int)pool->pages;
  return r;
}

}  // namespace clm

using namespace clm;

struct clm_b200_pages {
  PageLedger ledger;
  explicit clm_b200_pages(uint32_t n) : ledger(n) {}
};

namespace {

bool aligned16(const void* p, long long ld, size_t es) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (uint64_t)ld * es % 16 == 0;
}

template <typename S, typename T>
int launch_append(const AppendArgs& a, cudaStream_t st) {
  const size_t smem = (size_t)kAppendRows * (a.rot / 2) * sizeof(float2) + (size_t)a.heads * kAppendRows * (a.hd + 2) * sizeof(T);
  CLM_TRY(ensure_smem(kv_append_kernel<S, T>, smem + kAppendRows * sizeof(int)));  // (the limit counts static memory too)
  return launch_pdl(kv_append_kernel<S, T>, dim3((unsigned)(a.seqs.n * a.blocks), (unsigned)ceil_div(a.nkv, a.heads)),
                    dim3(kAppendThreads), smem, st, a);
}

}  // namespace

extern "C" {

int clm_b200_kv_append(clm_b200_ctx* ctx, const clm_b200_kv_pool* pool, uint32_t layer, const clm_b200_kv_seqs* seqs,
                       uint32_t n, uint32_t positions, uint32_t n_heads, int src_dtype, const void* d_q, uint64_t ld_q,
                       const void* d_k, uint64_t ld_k, const void* d_v, uint64_t ld_v, const clm_b200_rope* rope,
                       const int32_t* d_parents, void* d_q_out, void* stream) {
  CLM_CHECK(ctx != nullptr, CLM_INVALID_ARGUMENT, "null context");
  CLM_TRY(check_kv_pool(pool));
  CLM_TRY(check_kv_seqs(seqs));
  CLM_CHECK(layer < pool->layers, CLM_OUT_OF_RANGE, "layer outside the pool");
  CLM_CHECK(n <= seqs->rows, CLM_OUT_OF_RANGE, "more sequences than page tables");
  CLM_CHECK(n_heads == 0 || n_heads % pool->n_kv_heads == 0, CLM_INVALID_ARGUMENT,
            "query heads must be a multiple of the kv heads");
  CLM_CHECK(src_dtype >= CLM_DTYPE_F32 && src_dtype <= CLM_DTYPE_BF16, CLM_INVALID_ARGUMENT, "unknown element type");
  const uint32_t rot = rope ? rope->rot : 0;
  if (rope) {
    CLM_CHECK(rope->layout == CLM_ROPE_INTERLEAVED || rope->layout == CLM_ROPE_HALF, CLM_INVALID_ARGUMENT,
              "unknown rotary layout");
    CLM_CHECK(rot % 2 == 0 && rot <= pool->head_dim, CLM_INVALID_ARGUMENT,
              "the rotated part must be an even number of dims of the head");
    CLM_CHECK(rot == 0 || rope->d_inv_freq != nullptr, CLM_INVALID_ARGUMENT, "null frequencies");
  }
  if (n == 0 || positions == 0) return CLM_OK;
  CLM_CHECK(d_k && d_v && (!d_q || (d_q_out && n_heads > 0)), CLM_INVALID_ARGUMENT, "null buffer");
  CLM_CHECK(positions <= (1u << 24) && (uint64_t)n * positions <= 0x7fffffffull, CLM_OUT_OF_RANGE, "too many rows");
  CLM_CHECK(d_parents == nullptr || positions <= (uint32_t)kKvMaxWindow, CLM_OUT_OF_RANGE,
            "a tree window has at most 256 nodes");
  const uint64_t kd = (uint64_t)pool->n_kv_heads * pool->head_dim, qd = (uint64_t)n_heads * pool->head_dim;
  CLM_CHECK(ld_k >= kd && ld_v >= kd && (!d_q || ld_q >= qd) && std::max(ld_q, std::max(ld_k, ld_v)) < (1ull << 40),
            CLM_INVALID_ARGUMENT, "a row stride is smaller than a row");
  CLM_CHECK((uint64_t)n * positions - 1 <= (1ull << 58) / std::max(d_q ? ld_q : 1, std::max(ld_k, ld_v)), CLM_OUT_OF_RANGE,
            "the rows do not fit into an address space");
  CLM_CHECK(!d_q || (reinterpret_cast<uintptr_t>(d_q_out) & 15) == 0, CLM_INVALID_ARGUMENT,
            "the rotated queries must be 16-byte aligned");
  if (d_q) {  // rotated pairs are read by several threads, and the kv heads' CTAs write while others read
    const uint64_t rows = (uint64_t)n * positions, o = reinterpret_cast<uintptr_t>(d_q_out);
    auto apart = [&](const void* p, uint64_t ld, uint64_t row) {
      const uint64_t at = reinterpret_cast<uintptr_t>(p);
      return o >= at + ((rows - 1) * ld + row) * dtype_size(src_dtype) || at >= o + rows * qd * 2;
    };
    CLM_CHECK(apart(d_q, ld_q, qd) && apart(d_k, ld_k, kd) && apart(d_v, ld_v, kd), CLM_INVALID_ARGUMENT,
              "the rotated queries must not overlap the rows");
  }
  AppendArgs a{};
  a.seqs = make_kv_seqs(pool, seqs, n);
  const uint64_t off = (uint64_t)layer * pool->pages * kv_page_bytes(pool);
  a.q = d_q;
  a.k = d_k;
  a.v = d_v;
  a.ld_q = (long long)ld_q;
  a.ld_k = (long long)ld_k;
  a.ld_v = (long long)ld_v;
  a.q_out = d_q_out;
  a.kpool = static_cast<uint8_t*>(pool->k) + off;
  a.vpool = static_cast<uint8_t*>(pool->v) + off;
  a.freq = rope ? rope->d_inv_freq : nullptr;
  a.scale = rope ? rope->scale : 1.0f;
  a.parent = d_parents;
  a.positions = (int)positions;
  a.nh = n_heads ? (int)n_heads : (int)pool->n_kv_heads;
  a.nkv = (int)pool->n_kv_heads;
  a.hd = (int)pool->head_dim;
  a.rot = (int)rot;
  a.interleaved = rope && rope->layout == CLM_ROPE_INTERLEAVED;
  // blocks that `positions` rows starting anywhere touch at most
  a.blocks = positions == 1 ? 1 : (int)((positions - 2) / kAppendRows + 2);
  CLM_CHECK((uint64_t)n * a.blocks <= 0x7fffffffull, CLM_OUT_OF_RANGE, "too many rows");
  // As few splits of the kv heads as fill the GPU (the angles are evaluated in each).
  uint64_t splits = ceil_div((uint64_t)a.nkv, kAppendHeads);
  splits = std::max(splits, std::min((uint64_t)a.nkv, ceil_div(6ull * ctx->sm_count, (uint64_t)n * a.blocks)));
  a.heads = (int)ceil_div((uint64_t)a.nkv, splits);
  const size_t es = dtype_size(src_dtype);
  a.vec_q = aligned16(d_q, a.ld_q, es);
  a.vec_k = aligned16(d_k, a.ld_k, es);
  a.vec_v = aligned16(d_v, a.ld_v, es);
  CLM_SCOPE(ctx);
  cudaStream_t st = pick_stream(ctx, stream);
  const bool h = pool->dtype == CLM_DTYPE_F16;
  switch (src_dtype) {
    case CLM_DTYPE_F32:
      return h ? launch_append<float, __half>(a, st) : launch_append<float, __nv_bfloat16>(a, st);
    case CLM_DTYPE_F16:
      return h ? launch_append<__half, __half>(a, st) : launch_append<__half, __nv_bfloat16>(a, st);
    default:
      return h ? launch_append<__nv_bfloat16, __half>(a, st) : launch_append<__nv_bfloat16, __nv_bfloat16>(a, st);
  }
}

int clm_b200_rope_frequencies(int kind, uint32_t rot, double theta, double factor, double low, double high,
                              double original, double* h_inv_freq, float* h_scale) {
  CLM_CHECK(h_inv_freq != nullptr && h_scale != nullptr, CLM_INVALID_ARGUMENT, "null output");
  CLM_CHECK(rot >= 2 && rot % 2 == 0 && theta > 1.0 && std::isfinite(theta), CLM_INVALID_ARGUMENT,
            "an even number of rotated dims and a base above 1");
  CLM_CHECK(kind >= CLM_ROPE_PLAIN && kind <= CLM_ROPE_YARN, CLM_INVALID_ARGUMENT, "unknown frequency scaling");
  CLM_CHECK(kind == CLM_ROPE_PLAIN || (factor >= 1.0 && std::isfinite(factor)), CLM_INVALID_ARGUMENT,
            "a scaling factor is at least 1");
  CLM_CHECK(kind < CLM_ROPE_BANDS || (original > 0.0 && std::isfinite(original) && low > 0.0 && high > low),
            CLM_INVALID_ARGUMENT, "the bands need the original context and 0 < low < high");
  const double two_pi = 6.283185307179586;
  // YaRN (Peng et al. 2023): pair index at which the original context holds r turns
  auto pair_of = [&](double r) { return rot * std::log(original / (r * two_pi)) / (2.0 * std::log(theta)); };
  *h_scale = kind == CLM_ROPE_YARN ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
  for (uint32_t j = 0; j < rot / 2; ++j) {
    const double f = std::pow(theta, -2.0 * j / rot);
    double keep = 1.0;  // 1: the frequency as it is, 0: divided by the factor
    if (kind == CLM_ROPE_LINEAR) keep = 0.0;
    if (kind == CLM_ROPE_BANDS) keep = std::min(1.0, std::max(0.0, (original * f / two_pi - low) / (high - low)));
    if (kind == CLM_ROPE_YARN) {
      const double a = std::max(0.0, std::floor(pair_of(high)));
      const double b = std::min((double)rot - 1.0, std::ceil(pair_of(low)));
      keep = 1.0 - std::min(1.0, std::max(0.0, (j - a) / std::max(b - a, 0.001)));
    }
    h_inv_freq[j] = keep * f + (1.0 - keep) * f / (kind == CLM_ROPE_PLAIN ? 1.0 : factor);
  }
  return CLM_OK;
}

int clm_b200_kv_fork(clm_b200_ctx* ctx, const clm_b200_kv_pool* pool, const clm_b200_kv_seqs* seqs, uint32_t n,
                     const uint32_t* h_parents, const uint32_t* h_children, const int32_t* h_new_pages, void* stream) {
  CLM_CHECK(ctx != nullptr, CLM_INVALID_ARGUMENT, "null context");
  CLM_TRY(check_kv_pool(pool));
  CLM_TRY(check_kv_seqs(seqs));
  if (n == 0) return CLM_OK;
  CLM_CHECK(h_parents && h_children && h_new_pages, CLM_INVALID_ARGUMENT, "null argument");
  CLM_CHECK(n <= (uint32_t)kKvCopyMax, CLM_OUT_OF_RANGE, "at most 256 forks a call");
  CLM_CHECK(seqs->rows <= 65536, CLM_OUT_OF_RANGE, "at most 65536 page tables");
  for (uint32_t i = 0; i < n; ++i) {
    CLM_CHECK(h_parents[i] < seqs->rows && h_children[i] < seqs->rows, CLM_OUT_OF_RANGE, "no such page table");
    CLM_CHECK(h_new_pages[i] >= 0 && (uint32_t)h_new_pages[i] < pool->pages, CLM_OUT_OF_RANGE, "page outside the pool");
  }
  {
    uint32_t kids[kKvCopyMax];
    std::copy(h_children, h_children + n, kids);
    std::sort(kids, kids + n);
    CLM_CHECK(std::adjacent_find(kids, kids + n) == kids + n, CLM_INVALID_ARGUMENT, "a child appears twice");
    for (uint32_t i = 0; i < n; ++i)
      CLM_CHECK(!std::binary_search(kids, kids + n, h_parents[i]), CLM_INVALID_ARGUMENT,
                "a sequence is parent and child of one call");
    int32_t pages[kKvCopyMax];
    std::copy(h_new_pages, h_new_pages + n, pages);
    std::sort(pages, pages + n);
    CLM_CHECK(std::adjacent_find(pages, pages + n) == pages + n, CLM_INVALID_ARGUMENT, "a page appears twice");
  }
  CLM_SCOPE(ctx);
  ForkJob job;
  job.n = (int)n;
  for (uint32_t i = 0; i < n; ++i) {
    job.parent[i] = (uint16_t)h_parents[i];
    job.child[i] = (uint16_t)h_children[i];
    job.page[i] = h_new_pages[i];
  }
  const uint64_t pb = kv_page_bytes(pool);
  const SlabArgs s{static_cast<uint8_t*>(pool->k), static_cast<uint8_t*>(pool->v), pb * pool->pages, pb, pool->layers};
  const unsigned grid = std::max(copy_grid(pb, pool->layers, (int)n, ctx->sm_count), std::min(n, 1024u));
  return launch_pdl(kv_fork_kernel, dim3(grid), dim3(kCopyThreads), 0, pick_stream(ctx, stream), s, job, seqs->d_tables,
                    (int)seqs->max_pages, (int)pool->pages, reinterpret_cast<long long*>(seqs->d_pos));
}

int clm_b200_kv_copy_pages(clm_b200_ctx* ctx, const clm_b200_kv_pool* pool, uint32_t n, const int32_t* h_src,
                           const int32_t* h_dst, int32_t* d_tables, uint64_t table_entries, void* stream) {
  CLM_CHECK(ctx != nullptr, CLM_INVALID_ARGUMENT, "null context");
  CLM_TRY(check_kv_pool(pool));
  if (n == 0) return CLM_OK;
  CLM_CHECK(h_src && h_dst, CLM_INVALID_ARGUMENT, "null argument");
  for (uint32_t i = 0; i < n; ++i)
    CLM_CHECK(h_src[i] >= 0 && (uint32_t)h_src[i] < pool->pages && h_dst[i] >= 0 && (uint32_t)h_dst[i] < pool->pages,
              CLM_OUT_OF_RANGE, "page outside the pool");
  std::vector<std::pair<int32_t, int32_t>> pairs;
  std::vector<int32_t> dst;
  try {
    pairs.resize(n);
    dst.assign(h_dst, h_dst + n);
  } catch (const std::bad_alloc&) {
    return fail(CLM_RESOURCE_EXHAUSTED, "out of host memory");
  }
  for (uint32_t i = 0; i < n; ++i) pairs[i] = {h_src[i], h_dst[i]};
  std::sort(pairs.begin(), pairs.end());
  std::sort(dst.begin(), dst.end());
  CLM_CHECK(std::adjacent_find(dst.begin(), dst.end()) == dst.end(), CLM_INVALID_ARGUMENT, "a destination appears twice");
  for (uint32_t i = 0; i < n; ++i) {
    CLM_CHECK(!std::binary_search(dst.begin(), dst.end(), pairs[i].first), CLM_INVALID_ARGUMENT,
              "a page is source and destination of one call");
    CLM_CHECK(d_tables == nullptr || i == 0 || pairs[i].first != pairs[i - 1].first, CLM_INVALID_ARGUMENT,
              "a moved page has one destination");
  }
  CLM_SCOPE(ctx);
  const uint64_t pb = kv_page_bytes(pool);
  cudaStream_t st = pick_stream(ctx, stream);
  KvCopyJob job;
  for (uint32_t at = 0; at < n; at += kKvCopyMax) {
    job.n = (int)std::min<uint32_t>(kKvCopyMax, n - at);
    for (int i = 0; i < job.n; ++i) {
      job.src[i] = pairs[at + i].first;
      job.dst[i] = pairs[at + i].second;
    }
    CLM_TRY(launch_kv_copy(pool->k, pool->v, pool->layers, pb * pool->pages, pb, job, d_tables, table_entries,
                           ctx->sm_count, st));
  }
  return CLM_OK;
}

int clm_b200_pages_create(uint32_t pages, clm_b200_pages** out) {
  CLM_CHECK(out != nullptr, CLM_INVALID_ARGUMENT, "null output");
  *out = nullptr;
  CLM_CHECK(pages >= 1 && pages <= 0x7fffffffu, CLM_INVALID_ARGUMENT, "a pool has 1 to 2^31 - 1 pages");
  try {
    *out = new clm_b200_pages(pages);
  } catch (const std::bad_alloc&) {
    return fail(CLM_RESOURCE_EXHAUSTED, "out of host memory");
  }
  return CLM_OK;
}

int clm_b200_pages_destroy(clm_b200_pages* p) {
  delete p;
  return CLM_OK;
}

int clm_b200_pages_alloc(clm_b200_pages* p, uint32_t n, int32_t* h_ids) {
  CLM_CHECK(p != nullptr && (n == 0 || h_ids != nullptr), CLM_INVALID_ARGUMENT, "null argument");
  CLM_CHECK(p->ledger.alloc(n, h_ids), CLM_RESOURCE_EXHAUSTED,
            "only " + std::to_string(p->ledger.free_count()) + " pages are free");
  return CLM_OK;
}

int clm_b200_pages_retain(clm_b200_pages* p, uint32_t n, const int32_t* h_ids) {
  CLM_CHECK(p != nullptr && (n == 0 || h_ids != nullptr), CLM_INVALID_ARGUMENT, "null argument");
  for (uint32_t i = 0; i < n; ++i)
    CLM_CHECK(p->ledger.valid(h_ids[i]) && p->ledger.refs(h_ids[i]) > 0, CLM_NOT_FOUND, "page is not in use");
  for (uint32_t i = 0; i < n; ++i) p->ledger.retain(h_ids[i]);
  return CLM_OK;
}

int clm_b200_pages_release(clm_b200_pages* p, uint32_t n, const int32_t* h_ids) {
  CLM_CHECK(p != nullptr && (n == 0 || h_ids != nullptr), CLM_INVALID_ARGUMENT, "null argument");
  for (uint32_t i = 0; i < n; ++i) {
    // as many references as the list names the page: nothing is dropped when one is missing
    bool ok = p->ledger.valid(h_ids[i]) && p->ledger.refs(h_ids[i]) > 0;
    if (ok) {
      p->ledger.release(h_ids[i]);
      continue;
    }
    for (uint32_t j = i; j-- > 0;) p->ledger.restore(h_ids[j]);
    return fail(CLM_NOT_FOUND, "page is not in use");
  }
  return CLM_OK;
}

int clm_b200_pages_info(const clm_b200_pages* p, int32_t id, uint32_t* h_refs, uint32_t* h_free) {
  CLM_CHECK(p != nullptr, CLM_INVALID_ARGUMENT, "null argument");
  if (h_refs != nullptr) {
    CLM_CHECK(p->ledger.valid(id), CLM_OUT_OF_RANGE, "page outside the pool");
    *h_refs = p->ledger.refs(id);
  }
  if (h_free != nullptr) *h_free = p->ledger.free_count();
  return CLM_OK;
}

int clm_b200_pages_compact(clm_b200_pages* p, uint32_t capacity, int32_t* h_src, int32_t* h_dst, uint32_t* h_moves) {
  CLM_CHECK(p != nullptr && h_moves != nullptr && (capacity == 0 || (h_src && h_dst)), CLM_INVALID_ARGUMENT,
            "null argument");
  uint32_t need = 0;
  for (uint32_t i = p->ledger.pages() - p->ledger.free_count(); i < p->ledger.pages(); ++i)
    need += p->ledger.refs(i) > 0;
  *h_moves = need;
  CLM_CHECK(need <= capacity, CLM_RESOURCE_EXHAUSTED, "the plan has " + std::to_string(need) + " moves");
  try {
    std::vector<int32_t> src, dst;
    src.reserve(need);
    dst.reserve(need);
    p->ledger.compact(src, dst);
    std::copy(src.begin(), src.end(), h_src);
    std::copy(dst.begin(), dst.end(), h_dst);
  } catch (const std::bad_alloc&) {
    return fail(CLM_RESOURCE_EXHAUSTED, "out of host memory");
  }
  return CLM_OK;
}

}  // extern "C"
