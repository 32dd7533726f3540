// kv_attention.cu — attention of many sequences over a paged cache, shared leading pages read once.
//
// o = sum_j softmax_j(scale q . k_j) v_j over the positions j a row sees.  A row's positions fall into the pages that
// its sequence shares with its group and the sequence's own pages; both parts (and any further split of them) give a
// partial (unnormalised o, running maximum m, sum l), and partials combine by their maxima.
//
// Work is the list of (row tile, page) pairs.  An "entry" is a group's shared pages (rows: all query heads of a kv
// head of all the group's window rows) or a sequence's own pages (rows: its own); an entry has one item per (kv head,
// tile of up to 128 rows), and an item has as many work units as the entry has pages.  The line of all units is cut
// into equal shares, one per CTA, so ragged lengths balance without any host knowledge of them; a CTA's part of an item
// is a segment, and (item + CTA) numbers the segments without gaps to search.  A second kernel combines each row's
// segments.
//
// A CTA streams its units' pages through a ring of page slots (one producer warp, bulk copies); eight consumer warps
// split a page by row tiles of 16 and, when there are fewer than eight of these, by halves of the page and by pages.
#include <algorithm>
#include <cfloat>

#include "bulk.cuh"
#include "kv_ops.cuh"
#include "pdl.cuh"

namespace clm {

namespace {

constexpr int kMaxEntries = kKvMaxGroups + kKvMaxSeqs;
constexpr int kRowTile = 128;  // rows of an item: eight m16 tiles
constexpr int kWarps = 8;      // consumer warps
constexpr int kSegPad = 4;     // floats after a partial row's hd outputs: m, l, padding to 16 bytes

struct Plan {
  long long cum[kMaxEntries + 1];  // work units before entry e
  int pages[kMaxEntries];          // pages of an item of entry e
  int entries;
};

struct Args {
  KvSeqs seqs;
  KvGroups groups;
  const void *q, *k, *v;
  long long ld_q;
  void* out;
  const int32_t* parent;
  int positions, nh, nkv, group;
  float scale_log2;
  Plan* plan;
  float* part_g;  // segments of group items: [group items + CTAs][kRowTile][hd + kSegPad]
  float* part_s;  // segments of sequence items: [sequence items + CTAs][rows_s][hd + kSegPad]
  int rows_s;     // row capacity of a sequence item (16, 32, 64 or 128)
  int tiles_s;    // row tiles of a sequence
};

__host__ __device__ inline int tile_mt(int rows) { return rows <= 16 ? 1 : rows <= 32 ? 2 : rows <= 64 ? 4 : 8; }

// What entry e covers: groups first, then sequences.
struct Entry {
  int s0, s1;      // sequences
  int rows;        // rows per kv head
  int tiles;       // row tiles per kv head
  int first_page;  // first table entry
};
__device__ __forceinline__ Entry entry_of(const Args& a, int e) {
  Entry r;
  if (e < a.groups.n) {
    r.s0 = a.groups.start[e];
    r.s1 = a.groups.start[e + 1];
    r.first_page = 0;
    r.rows = (r.s1 - r.s0) * a.positions * a.group;
    r.tiles = (r.rows + kRowTile - 1) / kRowTile;
  } else {
    r.s0 = e - a.groups.n;
    r.s1 = r.s0 + 1;
    r.rows = a.positions * a.group;
    r.tiles = a.tiles_s;
    r.first_page = 0;
  }
  return r;
}

// The group of sequence b, or -1.
__device__ __forceinline__ int group_of(const Args& a, int b) {
  if (a.groups.n == 0 || b >= a.groups.start[a.groups.n]) return -1;
  int lo = 0, hi = a.groups.n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (a.groups.start[mid] <= b)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ int shared_pages(const Args& a, int b) {
  const int g = group_of(a, b);
  return g < 0 ? 0 : min((int)a.groups.pages[g], a.seqs.max_pages);
}

// Items before entry e, within its kind (groups, sequences).
__device__ __forceinline__ int items_before(const Args& a, int e) {
  if (e >= a.groups.n) return (e - a.groups.n) * a.tiles_s * a.nkv;
  int n = 0;
  for (int g = 0; g < e; ++g)
    n += ((a.groups.start[g + 1] - a.groups.start[g]) * a.positions * a.group + kRowTile - 1) / kRowTile * a.nkv;
  return n;
}

// The CTA whose share [c W / C, (c + 1) W / C) holds unit w.
__device__ __forceinline__ int cta_of(long long w, long long W, int C) {
  return (int)(((w + 1) * C + W - 1) / W) - 1;
}

// Fills `plan` from the device-side positions: pages per item, then the running work of the entries.
__device__ void make_plan(const Args& a, Plan* plan) {
  const int E = a.groups.n + a.seqs.n;
  for (int e = threadIdx.x; e < E; e += blockDim.x) {
    long long pages = 0, items;
    const Entry en = entry_of(a, e);
    items = (long long)en.tiles * a.nkv;
    if (e < a.groups.n) {
      pages = min((int)a.groups.pages[e], a.seqs.max_pages);
    } else {
      const long long base = a.seqs.base(en.s0);
      if (base >= 0) {
        pages = (base + a.positions + kPageTokens - 1) / kPageTokens;
        pages = min(pages, (long long)a.seqs.max_pages) - shared_pages(a, en.s0);
        if (pages < 0) pages = 0;
      }
    }
    plan->pages[e] = (int)pages;
    plan->cum[e + 1] = pages * items;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    long long run = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int e = e0 + threadIdx.x;
      long long x = e < E ? plan->cum[e + 1] : 0;
      for (int d = 1; d < 32; d <<= 1) {
        const long long o = __shfl_up_sync(0xffffffffu, x, d);
        if ((int)threadIdx.x >= d) x += o;
      }
      if (e < E) plan->cum[e + 1] = run + x;
      run += __shfl_sync(0xffffffffu, x, 31);
    }
    if (threadIdx.x == 0) {
      plan->cum[0] = 0;
      plan->entries = E;
    }
  }
  __syncthreads();
}

template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Pairs of 16-bit values with an all-ones exponent (infinities, NaN): the exponent's mask, and 1.0.
template <typename T>
constexpr uint32_t kExpMask = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
template <typename T>
constexpr uint32_t kOne = std::is_same<T, __half>::value ? 0x3C00u : 0x3F80u;

template <typename T>
__device__ __forceinline__ bool has_nonfinite(uint32_t w) {
  return (w & kExpMask<T>) == kExpMask<T> || ((w >> 16) & kExpMask<T>) == kExpMask<T>;
}
template <typename T>
__device__ __forceinline__ uint32_t nonfinite_mask(uint32_t w) {  // 0xffff at each non-finite half
  return ((w & kExpMask<T>) == kExpMask<T> ? 0xffffu : 0u) |
         (((w >> 16) & kExpMask<T>) == kExpMask<T> ? 0xffff0000u : 0u);
}

template <int HD>
struct Tile {
  static constexpr uint32_t kPage = kPageTokens * HD * 2;  // bytes of K, or V, of one page and kv head
  static constexpr int kSlots = HD == 128 ? 4 : 8;
  static constexpr int kRow = HD + kSegPad;
  static constexpr size_t kSmem = (size_t)kSlots * 2 * kPage + (size_t)kWarps * 16 * kRow * sizeof(float);
};

__device__ __forceinline__ void mbar_arrive_n(uint64_t* bar, uint32_t n) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_addr(bar)), "r"(n) : "memory");
}
__device__ __forceinline__ void consumer_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory"); }

// Whether window row i sees window row j: j's bit in i's ancestor set, or the chain's j <= i.
struct Window {
  const uint32_t* anc;  // [positions][8] bits in shared memory, or null
  int positions;
  __device__ __forceinline__ bool sees(int i, long long j) const {
    if (j >= positions) return false;
    return anc ? (anc[8 * i + (int)(j >> 5)] >> (j & 31)) & 1u : j <= i;
  }
};

template <typename T, int HD>
__global__ void __launch_bounds__(32 * (kWarps + 1), 1) kv_attention_kernel(const __grid_constant__ Args a) {
  using TL = Tile<HD>;
  constexpr int KW = HD / 32;  // 16-byte words of a K row per lane
  extern __shared__ __align__(128) uint8_t at_smem[];
  __shared__ Plan plan;
  __shared__ __align__(8) uint64_t full[TL::kSlots], empty[TL::kSlots];
  __shared__ int s_page[TL::kSlots];
  __shared__ uint32_t s_anc[kKvMaxWindow * 8];
  float* parts = reinterpret_cast<float*>(at_smem + (size_t)TL::kSlots * 2 * TL::kPage);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  if (threadIdx.x == 0) {
    for (int s = 0; s < TL::kSlots; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], kWarps);
    }
    mbar_fence_init();
  }
  griddep_wait();
  griddep_launch();
  make_plan(a, &plan);
  if (a.parent != nullptr) {  // ancestor sets of the tree's nodes
    for (int i = threadIdx.x; i < a.positions; i += blockDim.x) {
      uint32_t bits[8] = {};
      for (int at = i;;) {
#pragma unroll
        for (int w = 0; w < 8; ++w)
          if (w == at >> 5) bits[w] |= 1u << (at & 31);
        const int up = a.parent[at];
        if (up < 0 || up >= at) break;
        at = up;
      }
#pragma unroll
      for (int w = 0; w < 8; ++w) s_anc[8 * i + w] = bits[w];
    }
  }
  if (blockIdx.x == 0)  // the combining kernel's copy
    for (int i = threadIdx.x; i < (int)(sizeof(Plan) / 4); i += blockDim.x)
      reinterpret_cast<int*>(a.plan)[i] = reinterpret_cast<const int*>(&plan)[i];
  __syncthreads();
  const int E = plan.entries;
  const long long W = plan.cum[E];
  const int C = (int)min((long long)gridDim.x, W);  // every share holds a unit
  if ((int)blockIdx.x >= C) return;
  const long long w_begin = (long long)blockIdx.x * W / C, w_end = (long long)(blockIdx.x + 1) * W / C;
  int e = 0;  // the entry of the first unit
  {
    int lo = 0, hi = E - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (plan.cum[mid] <= w_begin)
        lo = mid;
      else
        hi = mid - 1;
    }
    e = lo;
  }

  if (warp == kWarps) {
    // ---------------- producer ----------------
    int slot = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (long long w = w_begin; w < w_end && ok;) {
      while (plan.cum[e + 1] <= w) ++e;
      const Entry en = entry_of(a, e);
      const int L = plan.pages[e];
      const int tile = (int)((w - plan.cum[e]) / L), off = (int)((w - plan.cum[e]) % L);
      const int np = (int)min((long long)(L - off), w_end - w);
      const int kvh = tile / en.tiles;
      const int first = (e < a.groups.n ? 0 : shared_pages(a, en.s0)) + off;
      const int32_t* table = a.seqs.table(en.s0) + first;
      for (int j0 = 0; j0 < np && ok; j0 += 32) {
        const int32_t mine = j0 + lane < np ? __ldg(table + j0 + lane) : -1;
        for (int j = 0; j < min(32, np - j0); ++j) {
          const int32_t page = __shfl_sync(0xffffffffu, mine, j);
          if (lane == 0) {
            ok = mbar_wait(&empty[slot], phase ^ 1u, nullptr);
            if (ok) {
              const bool real = page >= 0 && page < a.seqs.pool_pages;
              s_page[slot] = real;
              if (real) {
                uint8_t* dst = at_smem + (size_t)slot * 2 * TL::kPage;
                const size_t src = ((size_t)page * a.nkv + kvh) * TL::kPage;
                mbar_expect_tx(&full[slot], 2 * TL::kPage);
                bulk_g2s(dst, static_cast<const uint8_t*>(a.k) + src, TL::kPage, &full[slot]);
                bulk_g2s(dst + TL::kPage, static_cast<const uint8_t*>(a.v) + src, TL::kPage, &full[slot]);
              } else {
                mbar_arrive(&full[slot]);
              }
            }
          }
          ok = __shfl_sync(0xffffffffu, ok, 0);
          if (!ok) break;
          if (++slot == TL::kSlots) {
            slot = 0;
            phase ^= 1u;
          }
        }
      }
      w += np;
    }
    return;
  }

  // ---------------- consumers ----------------
  const int g = lane / 4, t = lane % 4;
  const Window win{a.parent ? s_anc : nullptr, a.positions};
  long long count = 0;  // pages of this CTA's stream so far: page i is in slot i % kSlots
  bool failed = false;
  for (long long w = w_begin; w < w_end;) {
    while (plan.cum[e + 1] <= w) ++e;
    const Entry en = entry_of(a, e);
    const bool is_group = e < a.groups.n;
    const int L = plan.pages[e];
    const int tile = (int)((w - plan.cum[e]) / L), off = (int)((w - plan.cum[e]) % L);
    const int np = (int)min((long long)(L - off), w_end - w);
    const int kvh = tile / en.tiles, x0 = (tile % en.tiles) * kRowTile;
    const int nrows = min(en.rows - x0, kRowTile);
    const int mt = tile_mt(nrows);
    const int first = (is_group ? 0 : shared_pages(a, en.s0)) + off;
    // this warp: row tile j, half (or both) of the pages of its turn
    const int j = warp % mt, kp = warp / mt;
    const int turns = mt == 1 ? 4 : mt == 2 ? 2 : 1, turn = mt <= 2 ? kp / 2 : 0;
    const int h_begin = mt == 8 ? 0 : kp % 2, h_end = mt == 8 ? 2 : h_begin + 1;
    const uint32_t arrivals = mt == 1 ? 4 : mt == 2 ? 2 : 1;

    // rows r0 = 16 j + g and r0 + 8 of the tile: window row and head
    int i0, i1;
    long long b0, b1;
    bool v0, v1;
    uint4 qw0[KW], qw1[KW];
    auto row = [&](int r, int& i, long long& base, bool& valid, uint4(&qw)[KW]) {
      const int x = x0 + r;
      valid = r < nrows;
      const int srow = valid ? x / a.group : 0, head = kvh * a.group + (valid ? x % a.group : 0);
      const int b = en.s0 + srow / a.positions;
      i = srow % a.positions;
      base = a.seqs.base(b);
      valid = valid && base >= 0;
      const uint4* p = reinterpret_cast<const uint4*>(
          static_cast<const T*>(a.q) + ((long long)b * a.positions + i) * a.ld_q + (long long)head * HD + (HD / 4) * t);
#pragma unroll
      for (int u = 0; u < KW; ++u) qw[u] = valid ? __ldg(p + u) : make_uint4(0u, 0u, 0u, 0u);
    };
    row(16 * j + g, i0, b0, v0, qw0);
    row(16 * j + g + 8, i1, b1, v1, qw1);
    auto word = [](const uint4(&v)[KW], int k) {
      const uint4& u = v[k / 4];
      return (k % 4 == 0) ? u.x : (k % 4 == 1) ? u.y : (k % 4 == 2) ? u.z : u.w;
    };
    float O[HD / 8][4];
#pragma unroll
    for (int n = 0; n < HD / 8; ++n) O[n][0] = O[n][1] = O[n][2] = O[n][3] = 0.0f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;

    for (int pj = 0; pj < np; ++pj, ++count) {
      if (turns > 1 && (pj & (turns - 1)) != turn) continue;
      const int slot = (int)(count % TL::kSlots);
      const bool arrived = !failed && mbar_wait(&full[slot], (uint32_t)(count / TL::kSlots) & 1u, nullptr);
      failed = !arrived;
      if (arrived && s_page[slot]) {
        const T* ks = reinterpret_cast<const T*>(at_smem + (size_t)slot * 2 * TL::kPage);
        const T* vs = ks + kPageTokens * HD;
        const long long p_begin = (long long)(first + pj) * kPageTokens;
        // every position visible to every valid row of the warp's tile (a row of no sequence sees nothing)
        const bool plain = __all_sync(0xffffffffu, (!v0 || p_begin + kPageTokens <= b0) && (!v1 || p_begin + kPageTokens <= b1));
        for (int half = h_begin; half < h_end; ++half) {
          float S[4][4];
#pragma unroll
          for (int jj = 0; jj < 4; ++jj) {
            S[jj][0] = S[jj][1] = S[jj][2] = S[jj][3] = 0.0f;
            const int pos = 32 * half + 8 * (g / 2) + 2 * jj + (g % 2);
            const uint4* kr = reinterpret_cast<const uint4*>(ks + (size_t)pos * HD);
            uint4 kw[KW];
#pragma unroll
            for (int u = 0; u < KW; ++u) kw[u] = kr[kv_k_chunk(KW * t + u, pos)];
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk)
              mma16<T>(S[jj], word(qw0, 2 * kk), word(qw1, 2 * kk), word(qw0, 2 * kk + 1), word(qw1, 2 * kk + 1),
                       word(kw, 2 * kk), word(kw, 2 * kk + 1));
          }
          uint32_t see = 0;  // masked pages: bit 4 jj + e of the positions a row sees
          float mx0 = m0, mx1 = m1;
#pragma unroll
          for (int jj = 0; jj < 4; ++jj)
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              bool s0 = v0, s1 = v1;
              if (!plain) {
                const long long pos = p_begin + 32 * half + 8 * t + 2 * jj + x;
                s0 = v0 && (pos < b0 || win.sees(i0, pos - b0));
                s1 = v1 && (pos < b1 || win.sees(i1, pos - b1));
                see |= (s0 ? 1u : 0u) << (4 * jj + x) | (s1 ? 1u : 0u) << (4 * jj + 2 + x);
              }
              S[jj][x] = s0 ? S[jj][x] * a.scale_log2 : -INFINITY;
              S[jj][2 + x] = s1 ? S[jj][2 + x] * a.scale_log2 : -INFINITY;
              mx0 = fmaxf(mx0, S[jj][x]);
              mx1 = fmaxf(mx1, S[jj][2 + x]);
            }
#pragma unroll
          for (int o = 1; o <= 2; o <<= 1) {
            mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, o));
            mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, o));
          }
          // a row that has seen nothing yet keeps m = -inf: its terms are exp2(-inf) through a zero reference
          const float r0 = mx0 == -INFINITY ? 0.0f : mx0, r1 = mx1 == -INFINITY ? 0.0f : mx1;
          const float c0 = exp2f(m0 - r0), c1 = exp2f(m1 - r1);
          m0 = mx0;
          m1 = mx1;
          l0 *= c0;
          l1 *= c1;
#pragma unroll
          for (int n = 0; n < HD / 8; ++n) {
            O[n][0] *= c0;
            O[n][1] *= c0;
            O[n][2] *= c1;
            O[n][3] *= c1;
          }
          uint32_t pa[4][2];
#pragma unroll
          for (int jj = 0; jj < 4; ++jj) {
            const float p00 = exp2f(S[jj][0] - r0), p01 = exp2f(S[jj][1] - r0);
            const float p10 = exp2f(S[jj][2] - r1), p11 = exp2f(S[jj][3] - r1);
            l0 += p00 + p01;  // this lane's positions; the quad's lanes add up at the end of the segment
            l1 += p10 + p11;
            pa[jj][0] = pack2<T>(p00, p01);
            pa[jj][1] = pack2<T>(p10, p11);
          }
#pragma unroll
          for (int n = 0; n < HD / 8; ++n) {
            const int vrow = 8 * n + g;
            uint4 va = reinterpret_cast<const uint4*>(vs + (size_t)vrow * kPageTokens)[kv_v_chunk(4 * half + t, vrow)];
            if (!plain) {
              // 0 * inf and 0 * NaN: a value that is not finite counts only for the rows that see its position.  Such
              // values are replaced by zero, and a second product of indicators finds the outputs they reach.
              const bool odd = has_nonfinite<T>(va.x) || has_nonfinite<T>(va.y) || has_nonfinite<T>(va.z) ||
                               has_nonfinite<T>(va.w);
              if (__any_sync(0xffffffffu, odd)) {
                const uint32_t bx = nonfinite_mask<T>(va.x), by = nonfinite_mask<T>(va.y), bz = nonfinite_mask<T>(va.z),
                               bw = nonfinite_mask<T>(va.w);
                uint32_t in[4][2];
#pragma unroll
                for (int jj = 0; jj < 4; ++jj)
#pragma unroll
                  for (int r = 0; r < 2; ++r)
                    in[jj][r] = ((see >> (4 * jj + 2 * r)) & 1u ? kOne<T> : 0u) |
                                ((see >> (4 * jj + 2 * r + 1)) & 1u ? kOne<T> << 16 : 0u);
                constexpr uint32_t one2 = kOne<T> | kOne<T> << 16;
                float hit[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                mma16<T>(hit, in[0][0], in[0][1], in[1][0], in[1][1], bx & one2, by & one2);
                mma16<T>(hit, in[2][0], in[2][1], in[3][0], in[3][1], bz & one2, bw & one2);
#pragma unroll
                for (int x = 0; x < 4; ++x)
                  if (hit[x] > 0.0f) O[n][x] = NAN;
                va = make_uint4(va.x & ~bx, va.y & ~by, va.z & ~bz, va.w & ~bw);
              }
            }
            mma16<T>(O[n], pa[0][0], pa[0][1], pa[1][0], pa[1][1], va.x, va.y);
            mma16<T>(O[n], pa[2][0], pa[2][1], pa[3][0], pa[3][1], va.z, va.w);
          }
        }
      }
      __syncwarp();
      if (lane == 0 && arrived) mbar_arrive_n(&empty[slot], arrivals);
    }
    w += np;

    // the warps that share a row tile fold their states; the segment's rows go to its partial
    float* sp = parts + (size_t)warp * 16 * TL::kRow;
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, o);
      l1 += __shfl_xor_sync(0xffffffffu, l1, o);
    }
    if (failed) l0 = l1 = NAN;  // a copy never arrived: the rows say so
#pragma unroll
    for (int n = 0; n < HD / 8; ++n) {
      *reinterpret_cast<float2*>(sp + g * TL::kRow + 8 * n + 2 * t) = make_float2(O[n][0], O[n][1]);
      *reinterpret_cast<float2*>(sp + (g + 8) * TL::kRow + 8 * n + 2 * t) = make_float2(O[n][2], O[n][3]);
    }
    if (t == 0) {
      sp[g * TL::kRow + HD] = m0;
      sp[g * TL::kRow + HD + 1] = l0;
      sp[(g + 8) * TL::kRow + HD] = m1;
      sp[(g + 8) * TL::kRow + HD + 1] = l1;
    }
    consumer_sync();
    const int seg = items_before(a, e) + tile + (int)blockIdx.x;
    float* dst = is_group ? a.part_g + (size_t)seg * kRowTile * TL::kRow : a.part_s + (size_t)seg * a.rows_s * TL::kRow;
    constexpr int C4 = HD / 4;
    for (int idx = threadIdx.x; idx < nrows * C4; idx += 32 * kWarps) {
      const int r = idx / C4, c4 = idx % C4;
      const float* src = parts + ((size_t)(r / 16) * 16 + r % 16) * TL::kRow;
      const size_t step = (size_t)mt * 16 * TL::kRow;
      float M = -INFINITY;
      for (int k = 0; k < kWarps / mt; ++k) M = fmaxf(M, src[k * step + HD]);
      const float R = M == -INFINITY ? 0.0f : M;
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      float l = 0.0f;
      for (int k = 0; k < kWarps / mt; ++k) {
        const float f = exp2f(src[k * step + HD] - R);
        const float4 o = *reinterpret_cast<const float4*>(src + k * step + 4 * c4);
        acc = make_float4(acc.x + o.x * f, acc.y + o.y * f, acc.z + o.z * f, acc.w + o.w * f);
        l += src[k * step + HD + 1] * f;
      }
      *reinterpret_cast<float4*>(dst + (size_t)r * TL::kRow + 4 * c4) = acc;
      if (c4 == 0) *reinterpret_cast<float2*>(dst + (size_t)r * TL::kRow + HD) = make_float2(M, l);
    }
    consumer_sync();
  }
}

// One warp per (row, head): the row's segments of its group's item and of its own, combined by their maxima.
template <typename T, int HD>
__global__ void __launch_bounds__(256) kv_combine_kernel(const __grid_constant__ Args a, int ctas) {
  using TL = Tile<HD>;
  constexpr int N = HD / 32;  // outputs per lane
  griddep_wait();
  griddep_launch();
  const int lane = threadIdx.x % 32;
  const long long id = (long long)blockIdx.x * 8 + threadIdx.x / 32;
  if (id >= (long long)a.seqs.n * a.positions * a.nh) return;
  const int head = (int)(id % a.nh), row = (int)(id / a.nh);
  const int b = row / a.positions, kvh = head / a.group;
  const Plan* plan = a.plan;
  const long long W = plan->cum[plan->entries];
  const int C = (int)min((long long)ctas, W);
  const bool idle = a.seqs.base(b) < 0;
  const int grp = idle ? -1 : group_of(a, b);
  float M = -INFINITY, l = 0.0f, acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.0f;
#pragma unroll
  for (int part = 0; part < 2; ++part) {
    const int e = part == 0 ? grp : a.groups.n + b;
    if (e < 0 || idle) continue;
    const int L = plan->pages[e];
    if (L == 0) continue;
    const Entry en = entry_of(a, e);
    const int x = (row - en.s0 * a.positions) * a.group + head % a.group;
    const int tile = kvh * en.tiles + x / kRowTile, r = x % kRowTile;
    const long long w = plan->cum[e] + (long long)tile * L;
    const int c0 = cta_of(w, W, C), c1 = cta_of(w + L - 1, W, C);
    const int item = items_before(a, e) + tile;
    for (int c = c0; c <= c1; ++c) {
      const float* src = part == 0 ? a.part_g + ((size_t)(item + c) * kRowTile + r) * TL::kRow
                                   : a.part_s + ((size_t)(item + c) * a.rows_s + r) * TL::kRow;
      const float2 ml = *reinterpret_cast<const float2*>(src + HD);
      float o[N];
      if constexpr (N == 4) {
        const float4 f = *reinterpret_cast<const float4*>(src + 4 * lane);
        o[0] = f.x, o[1] = f.y, o[2] = f.z, o[3] = f.w;
      } else {
        const float2 f = *reinterpret_cast<const float2*>(src + 2 * lane);
        o[0] = f.x, o[1] = f.y;
      }
      const float m = fmaxf(M, ml.x), R = m == -INFINITY ? 0.0f : m;
      const float f0 = exp2f(M - R), f1 = exp2f(ml.x - R);
      M = m;
      l = l * f0 + ml.y * f1;
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = acc[i] * f0 + o[i] * f1;
    }
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
  T* out = static_cast<T*>(a.out) + ((size_t)row * a.nh + head) * HD + N * lane;
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = acc[i] * inv;
  } else if constexpr (N == 4) {
    *reinterpret_cast<uint2*>(out) =
        make_uint2(pack2<T>(acc[0] * inv, acc[1] * inv), pack2<T>(acc[2] * inv, acc[3] * inv));
  } else {
    *reinterpret_cast<uint32_t*>(out) = pack2<T>(acc[0] * inv, acc[1] * inv);
  }
}

size_t al256(size_t n) { return (n + 255) & ~(size_t)255; }

struct Sizes {
  int rows_s, tiles_s;
  size_t plan, part_g, part_s;  // bytes
  size_t total() const { return plan + part_g + part_s; }
};

Sizes sizes_of(int n, int positions, int nh, int nkv, int hd, const KvGroups& groups, int sm_count) {
  Sizes s;
  const int group = nh / nkv, rows = positions * group;
  s.rows_s = rows >= kRowTile ? kRowTile : 16 * tile_mt(rows);
  s.tiles_s = (rows + kRowTile - 1) / kRowTile;
  size_t items_g = 0;
  for (int g = 0; g < groups.n; ++g)
    items_g += (size_t)((groups.start[g + 1] - groups.start[g]) * rows + kRowTile - 1) / kRowTile * nkv;
  const size_t items_s = (size_t)n * s.tiles_s * nkv, row = (size_t)(hd + kSegPad) * sizeof(float);
  s.plan = al256(sizeof(Plan));
  s.part_g = groups.n ? al256((items_g + sm_count) * kRowTile * row) : 0;
  s.part_s = al256((items_s + sm_count) * s.rows_s * row);
  return s;
}

template <typename T, typename O, int HD>
int launch_typed(const Args& a, int sm_count, cudaStream_t st) {
  using TL = Tile<HD>;
  CLM_TRY(ensure_smem(kv_attention_kernel<T, HD>, TL::kSmem));
  CLM_TRY(launch_pdl(kv_attention_kernel<T, HD>, dim3((unsigned)sm_count), dim3(32 * (kWarps + 1)), TL::kSmem, st, a));
  const long long rows = (long long)a.seqs.n * a.positions * a.nh;
  return launch_pdl(kv_combine_kernel<O, HD>, dim3((unsigned)ceil_div(rows, 8)), dim3(256), 0, st, a, sm_count);
}

}  // namespace

size_t kv_attention_work(int n, int positions, int nh, int nkv, int hd, const KvGroups& groups, int sm_count) {
  return sizes_of(n, positions, nh, nkv, hd, groups, sm_count).total();
}

int launch_kv_attention(const KvAttnArgs& in, cudaStream_t st) {
  const Sizes s = sizes_of(in.seqs.n, in.positions, in.nh, in.nkv, in.hd, in.groups, in.sm_count);
  CLM_CHECK(in.work != nullptr && in.work_bytes >= s.total(), CLM_RESOURCE_EXHAUSTED, "attention workspace too small");
  Args a;
  a.seqs = in.seqs;
  a.groups = in.groups;
  a.q = in.q;
  a.k = in.k;
  a.v = in.v;
  a.ld_q = in.ld_q;
  a.out = in.out;
  a.parent = in.parent;
  a.positions = in.positions;
  a.nh = in.nh;
  a.nkv = in.nkv;
  a.group = in.nh / in.nkv;
  a.scale_log2 = in.scale * 1.4426950408889634f;
  uint8_t* w = static_cast<uint8_t*>(in.work);
  a.plan = reinterpret_cast<Plan*>(w);
  a.part_g = reinterpret_cast<float*>(w + s.plan);
  a.part_s = reinterpret_cast<float*>(w + s.plan + s.part_g);
  a.rows_s = s.rows_s;
  a.tiles_s = s.tiles_s;
  const bool h = in.type == CLM_DTYPE_F16, f32 = in.out_type == CLM_DTYPE_F32;
  if (in.hd == 64) {
    if (h) return f32 ? launch_typed<__half, float, 64>(a, in.sm_count, st) : launch_typed<__half, __half, 64>(a, in.sm_count, st);
    return f32 ? launch_typed<__nv_bfloat16, float, 64>(a, in.sm_count, st)
               : launch_typed<__nv_bfloat16, __nv_bfloat16, 64>(a, in.sm_count, st);
  }
  CLM_CHECK(in.hd == 128, CLM_UNIMPLEMENTED, "head_dim 64 or 128");
  if (h) return f32 ? launch_typed<__half, float, 128>(a, in.sm_count, st) : launch_typed<__half, __half, 128>(a, in.sm_count, st);
  return f32 ? launch_typed<__nv_bfloat16, float, 128>(a, in.sm_count, st)
             : launch_typed<__nv_bfloat16, __nv_bfloat16, 128>(a, in.sm_count, st);
}

}  // namespace clm

using namespace clm;

namespace {

// The groups that share something (a group of one sequence, or of no pages, reads its pages as its own).
int make_groups(uint32_t n, uint32_t n_groups, const uint32_t* seqs, const uint32_t* pages, KvGroups* out) {
  CLM_CHECK(n_groups <= (uint32_t)kKvMaxGroups, CLM_OUT_OF_RANGE, "at most 64 groups");
  CLM_CHECK(n_groups == 0 || (seqs && pages), CLM_INVALID_ARGUMENT, "null groups");
  uint64_t at = 0;
  out->n = (int)n_groups;
  for (uint32_t g = 0; g < n_groups; ++g) {
    out->start[g] = (uint16_t)at;
    out->pages[g] = seqs[g] > 1 ? std::min(pages[g], 0x7fffffffu) : 0u;
    at += seqs[g];
    CLM_CHECK(at <= n, CLM_INVALID_ARGUMENT, "the groups hold more sequences than the call");
  }
  out->start[n_groups] = (uint16_t)at;
  return CLM_OK;
}

int check_shape(uint32_t n, uint32_t positions, uint32_t nh, uint32_t nkv, uint32_t hd) {
  CLM_CHECK(n <= (uint32_t)kKvMaxSeqs, CLM_OUT_OF_RANGE, "at most 512 sequences a call");
  CLM_CHECK(positions <= (uint32_t)kKvMaxWindow, CLM_OUT_OF_RANGE, "at most 256 rows a sequence");
  CLM_CHECK(nkv >= 1 && nh >= 1 && nh % nkv == 0, CLM_INVALID_ARGUMENT, "query heads must be a multiple of the kv heads");
  CLM_CHECK(nh <= 1024, CLM_OUT_OF_RANGE, "at most 1024 query heads");
  CLM_CHECK(hd == 64 || hd == 128, CLM_UNIMPLEMENTED, "head_dim 64 or 128");
  return CLM_OK;
}

}  // namespace

extern "C" {

int clm_b200_kv_attention_workspace(clm_b200_ctx* ctx, uint32_t n, uint32_t positions, uint32_t n_heads,
                                    uint32_t n_kv_heads, uint32_t head_dim, uint32_t n_groups,
                                    const uint32_t* h_group_seqs, const uint32_t* h_group_pages, uint64_t* bytes) {
  CLM_CHECK(ctx != nullptr && bytes != nullptr, CLM_INVALID_ARGUMENT, "null argument");
  CLM_TRY(check_shape(n, positions, n_heads, n_kv_heads, head_dim));
  KvGroups groups;
  CLM_TRY(make_groups(n, n_groups, h_group_seqs, h_group_pages, &groups));
  *bytes = n == 0 || positions == 0 ? 0
                                    : kv_attention_work((int)n, (int)positions, (int)n_heads, (int)n_kv_heads,
                                                        (int)head_dim, groups, ctx->sm_count);
  return CLM_OK;
}

int clm_b200_kv_attention(clm_b200_ctx* ctx, const clm_b200_kv_pool* pool, uint32_t layer,
                          const clm_b200_kv_seqs* seqs, uint32_t n, uint32_t positions, uint32_t n_heads,
                          const void* d_q, uint64_t ld_q, uint32_t n_groups, const uint32_t* h_group_seqs,
                          const uint32_t* h_group_pages, const int32_t* d_parents, float scale, void* d_out,
                          void* d_work, uint64_t work_bytes, void* stream) {
  CLM_CHECK(ctx != nullptr, CLM_INVALID_ARGUMENT, "null context");
  CLM_TRY(check_kv_pool(pool));
  CLM_TRY(check_kv_seqs(seqs));
  CLM_TRY(check_shape(n, positions, n_heads, pool->n_kv_heads, pool->head_dim));
  CLM_CHECK(layer < pool->layers, CLM_OUT_OF_RANGE, "layer outside the pool");
  CLM_CHECK(n <= seqs->rows, CLM_OUT_OF_RANGE, "more sequences than page tables");
  KvAttnArgs a;
  CLM_TRY(make_groups(n, n_groups, h_group_seqs, h_group_pages, &a.groups));
  if (n == 0 || positions == 0) return CLM_OK;
  CLM_CHECK(d_q && d_out && d_work, CLM_INVALID_ARGUMENT, "null buffer");
  CLM_CHECK(ld_q >= (uint64_t)n_heads * pool->head_dim && ld_q % 8 == 0 && ld_q < (1ull << 40), CLM_INVALID_ARGUMENT,
            "query rows: a stride of at least a row, a multiple of 8 elements");
  CLM_CHECK(((reinterpret_cast<uintptr_t>(d_q) | reinterpret_cast<uintptr_t>(d_out) |
              reinterpret_cast<uintptr_t>(d_work)) & 15) == 0,
            CLM_INVALID_ARGUMENT, "queries, outputs and workspace must be 16-byte aligned");
  a.seqs = make_kv_seqs(pool, seqs, n);
  const uint64_t off = (uint64_t)layer * pool->pages * kv_page_bytes(pool);
  a.k = static_cast<const uint8_t*>(pool->k) + off;
  a.v = static_cast<const uint8_t*>(pool->v) + off;
  a.q = d_q;
  a.ld_q = (long long)ld_q;
  a.out = d_out;
  a.parent = d_parents;
  a.positions = (int)positions;
  a.nh = (int)n_heads;
  a.nkv = (int)pool->n_kv_heads;
  a.hd = (int)pool->head_dim;
  a.type = a.out_type = pool->dtype;
  a.scale = scale;
  a.work = d_work;
  a.work_bytes = work_bytes;
  a.sm_count = ctx->sm_count;
  CLM_SCOPE(ctx);
  return launch_kv_attention(a, pick_stream(ctx, stream));
}

}  // extern "C"
