// kv_attention.cu — attention of many sequences over a paged cache, shared leading pages read once.
//
// o = sum_j softmax_j(scale q . k_j) v_j over the positions j a row sees.  A row's positions fall into the pages that
// its sequence shares with its group and the sequence's own pages; both parts (and any further split of them) give a
// partial (unnormalised o, running maximum m, sum l), and partials combine by their maxima.
//
// An "entry" is a group's shared pages (rows: all query heads of a kv head of all the group's window rows) or a
// sequence's own pages (rows: its own).  Entries of up to kStreamRows rows per kv head are bound by reading the
// pages: the stream kernel, whose warps load the operands of mma.sync straight from global memory.  Entries of more
// rows by products and softmax: the tile kernel, on the tensor cores' accumulators in TMEM.  All groups of a call
// go to one of the two, and all sequences; so a call is one or two launches and the combining one.
//
// Work of a kernel is one line of units: per entry, per item (kv head, and row tile in the tile kernel), its pages
// (tile kernel: counted double for more than 128 rows; stream kernel: half pages), and some units for an item's own
// start and end.  The line is cut into equal shares, one per CTA (stream kernel: per warp), so ragged lengths balance
// without any host knowledge of them.  A share's part of an item is a segment, numbered by (item + share): both only
// grow along the line.
//
// GPU time of a call (fp16, head_dim 128, 32 heads over 8 unless said): 4 sequences of about 1,000 positions 13 us; 8
// tree windows of 16 rows over 4,096 shared positions 34 us; 64 windows of 4 rows, 16,384 shared and about 500 own
// positions each, 138 us (tile kernel 83 us, 0.83 PFLOP/s; stream kernel 36 us, 3.7 TB/s; combining kernel 10 us);
// 256 rows over 8,192 positions (bf16) 102 us (0.72 PFLOP/s in the tile kernel); 64 sequences of 2,048 positions, 8
// rows a kv head, 95 us (5.6 TB/s).
#include <algorithm>
#include <cfloat>

#include "bulk.cuh"
#include "kv_ops.cuh"
#include "pdl.cuh"

namespace clm {

namespace {

constexpr int kMaxEntries = kKvMaxGroups + kKvMaxSeqs;
// Entries of up to this many rows per kv head: the stream kernel.  (Whole calls with 17 to 64 rows, stream kernel
// with up to four row tiles against tile kernel, head_dim 128: 8 sequences of 8,192 positions 72-118 against 62-65
// us, 64 of 2,048 134-247 against 123-146, 4 of 512 12-15 against 16-17; up to 16 rows the stream kernel: 8 x 8,192
// 58-60 us.)
constexpr int kStreamRows = 16;
constexpr int kStreamWarps = 8;  // warps of a stream CTA
constexpr int kRowTile = 256;    // rows of an item of the tile kernel: two tiles of 128
constexpr int kSegPad = 8;     // floats after a partial row's hd outputs: m, l, padding to 32 bytes
constexpr int kStreamSwitch = 2;  // stream kernel: a segment's start and end take as long as this many half pages
// Tile kernel: a segment's start and end take as long as this many units.  (8 tree windows of 16 rows over 4,096 shared
// positions, both kinds of entries in the tile kernel: 0 units 81 us, 6 39 us, 12 34 us.)
constexpr int kSwitch = 12;

struct Plan {
  uint32_t cum[kMaxEntries + 1];  // work units before entry e (below 2^32: two per page, which the host counts)
  int pages[kMaxEntries];         // pages of an item of entry e (stream kernel: half pages with a position that is seen)
  uint32_t shares, q, r;          // how the line is cut (below)
  __device__ __forceinline__ struct Shares cut() const;
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
  uint32_t polls;  // a wait of the tile kernel gives up after so many
  int* err;        // and then this flag is raised (or null)
  // partials of groups [0] and sequences [1]: segment x rows (tile kernel: 2 x 128, or 2 x rows, one half per stream)
  struct Kind {
    Plan* plan;     // of the kernel that has this kind
    float* part;    // [segments][rows][hd + kSegPad]
    int rows;       // row capacity of a segment, tile kernel: of half of one
    int tiles;      // row tiles of an item (sequences)
    int tile;       // 1: the tile kernel, 0: the stream kernel
  } kind[2];
};

// What entry e covers: groups first, then sequences.
struct Entry {
  int s0, s1;  // sequences
  int kind;    // 0: group, 1: sequence
  int rows;    // rows per kv head
  int tiles;   // row tiles per kv head
  int weight;  // work units of a page
  int over;    // and of an item besides its pages
};
__device__ __forceinline__ Entry entry_of(const Args& a, int e) {
  Entry r;
  r.kind = e >= a.groups.n;
  if (r.kind == 0) {
    r.s0 = a.groups.start[e];
    r.s1 = a.groups.start[e + 1];
  } else {
    r.s0 = e - a.groups.n;
    r.s1 = r.s0 + 1;
  }
  r.rows = (r.s1 - r.s0) * a.positions * a.group;
  const bool tile = a.kind[r.kind].tile;
  r.tiles = tile ? (r.rows + kRowTile - 1) / kRowTile : 1;
  r.weight = tile && r.rows > 128 ? 2 : 1;
  r.over = tile ? kSwitch : kStreamSwitch;
  return r;
}

// Pages of an item before its unit `u`.
__device__ __forceinline__ uint32_t pages_before(const Entry& e, uint32_t u) {
  return u <= (uint32_t)e.over ? 0u : (u - e.over + e.weight - 1) / e.weight;
}
__device__ __forceinline__ uint32_t units_of(const Entry& e, uint32_t pages) {
  return pages ? pages * e.weight + e.over : 0u;
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

// Items before entry e, within its kind (groups, sequences).
__device__ __forceinline__ int items_before(const Args& a, int e) {
  if (e >= a.groups.n) return (e - a.groups.n) * a.kind[1].tiles * a.nkv;
  if (!a.kind[0].tile) return e * a.nkv;
  int n = 0;
  for (int g = 0; g < e; ++g)
    n += ((a.groups.start[g + 1] - a.groups.start[g]) * a.positions * a.group + kRowTile - 1) / kRowTile * a.nkv;
  return n;
}

// W units in C shares of q or q + 1: the first r have one more.
struct Shares {
  uint32_t C, q, r;
  __device__ __forceinline__ uint32_t begin(uint32_t c) const { return c * q + min(c, r); }
  __device__ __forceinline__ uint32_t of(uint32_t w) const {  // the share that holds unit w
    const uint32_t wide = r * (q + 1);
    return w < wide ? w / (q + 1) : r + (w - wide) / q;
  }
};

__device__ __forceinline__ Shares Plan::cut() const { return Shares{shares, q, r}; }

// Fills the plan of the tile (or stream) kernel from the device-side positions: pages per item, then the running work
// of its entries (the other kernel's have none).  first: a sequence's first page of its own; of a group the sequence whose
// table names its pages, the first that is not idle (an idle one's table may name anything).
__device__ void make_plan(const Args& a, Plan* plan, int* first, int tile, uint32_t shares) {
  const int G = a.groups.n, E = G + a.seqs.n, per = tile ? 1 : 2, unit = kPageTokens / per;
  auto put = [&](int e, const Entry& en, int pages) {
    plan->pages[e] = pages;
    plan->cum[e + 1] = a.kind[en.kind].tile == tile ? units_of(en, pages) * (uint32_t)(en.tiles * a.nkv) : 0u;
  };
  for (int e = threadIdx.x; e < G; e += blockDim.x) first[e] = a.seqs.n;
  __syncthreads();
  for (int e = G + threadIdx.x; e < E; e += blockDim.x) {
    const Entry en = entry_of(a, e);
    const long long base = a.seqs.base(en.s0);
    const int g = group_of(a, en.s0), at = g < 0 ? 0 : min((int)a.groups.pages[g], a.seqs.max_pages);
    int pages = 0;
    if (base >= 0) {
      pages = max(0, (int)min((base + a.positions + unit - 1) / unit, (long long)per * a.seqs.max_pages) - per * at);
      if (g >= 0) atomicMin(&first[g], en.s0);
    }
    first[e] = at;
    put(e, en, pages);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < G; e += blockDim.x)
    put(e, entry_of(a, e), first[e] < a.seqs.n ? per * min((int)a.groups.pages[e], a.seqs.max_pages) : 0);
  __syncthreads();
  if (threadIdx.x < 32) {
    uint32_t run = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int e = e0 + threadIdx.x;
      uint32_t x = e < E ? plan->cum[e + 1] : 0;
      for (int d = 1; d < 32; d <<= 1) {
        const uint32_t o = __shfl_up_sync(0xffffffffu, x, d);
        if ((int)threadIdx.x >= d) x += o;
      }
      if (e < E) plan->cum[e + 1] = run + x;
      run += __shfl_sync(0xffffffffu, x, 31);
    }
    if (threadIdx.x == 0) {
      plan->cum[0] = 0;
      // Every share holds a unit.  Of the stream kernel three: a short segment spends more on its start and its partial
      // (GPU time of a call with 4 sequences of about 1,000 positions, 8 kv heads, head_dim 128, with at least 2, 3,
      // 4 or 6 units a share: 14.5, 12.9, 13.6, 16.4 us).
      plan->shares = min(shares, tile ? run : (run + 2) / 3);
      plan->q = run ? run / plan->shares : 0u;
      plan->r = run ? run % plan->shares : 0u;
    }
  }
  __syncthreads();
}

// The entry that holds unit w (the last one that begins at or before it), found by the warp's lanes together.
__device__ __forceinline__ int entry_at(const Plan& plan, int entries, uint32_t w) {
  const int lane = threadIdx.x % 32;
  int e = 0;
  for (int at = 0; at < entries; at += 32) {
    const uint32_t n = __popc(__ballot_sync(0xffffffffu, at + lane < entries && plan.cum[at + lane] <= w));
    e += n;
    if (n < 32) break;
  }
  return e - 1;
}

// The combining kernel's copy of the plan.
__device__ __forceinline__ void publish(const Args& a, const Plan& plan, int tile) {
  Plan* to = a.kind[1].tile == tile ? a.kind[1].plan : a.kind[0].plan;
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < (int)(sizeof(Plan) / 4); i += blockDim.x)
      reinterpret_cast<int*>(to)[i] = reinterpret_cast<const int*>(&plan)[i];
}

// Ancestor sets of the tree's nodes, eight words each (an entry that is not an earlier node ends a chain).
__device__ __forceinline__ void make_ancestors(const Args& a, uint32_t* anc) {
  for (int i = threadIdx.x; i < a.positions; i += blockDim.x) {
    uint32_t* bits = anc + 8 * i;
    for (int w = 0; w < 8; ++w) bits[w] = 0;
    for (int at = i;;) {
      bits[at >> 5] |= 1u << (at & 31);
      const int up = a.parent[at];
      if (up < 0 || up >= at) break;
      at = up;
    }
  }
}

// Pairs of 16-bit values with an all-ones exponent (infinities, NaN): the exponent's mask.
template <typename T>
constexpr uint32_t kExpMask = std::is_same<T, __half>::value ? 0x7C00u : 0x7F80u;
template <typename T>
__device__ __forceinline__ bool has_nonfinite(uint32_t w) {
  return (w & kExpMask<T>) == kExpMask<T> || ((w >> 16) & kExpMask<T>) == kExpMask<T>;
}
template <typename T>
__device__ __forceinline__ uint32_t nonfinite_mask(uint32_t w) {  // 0xffff at each non-finite half
  return ((w & kExpMask<T>) == kExpMask<T> ? 0xffffu : 0u) |
         (((w >> 16) & kExpMask<T>) == kExpMask<T> ? 0xffff0000u : 0u);
}
// A pair as numbers of the type that count what is not finite in a sum of up to 63: 1 for infinity, 64 for -infinity,
// 4096 for NaN (0 for finite values).
template <typename T>
__device__ __forceinline__ uint32_t nonfinite_code(uint32_t w) {
  constexpr bool kHalf = std::is_same<T, __half>::value;
  constexpr uint32_t one = kHalf ? 0x3C00u : 0x3F80u, c64 = kHalf ? 0x5400u : 0x4280u, c4096 = kHalf ? 0x6C00u : 0x4580u;
  auto code = [](uint32_t h) {
    return (h & 0x7fffu) < kExpMask<T> ? 0u : (h & 0x7fffu) > kExpMask<T> ? c4096 : h >> 15 ? c64 : one;
  };
  return code(w & 0xffffu) | code(w >> 16) << 16;
}

// ---- tensor-core primitives (kind::f16: f16 or bf16 operands, f32 accumulators in TMEM)
// K-major operand tiles with the 128-byte swizzle: rows of 64 elements, 8-row atoms of 1024 bytes, 16-byte chunk c of
// row r at chunk c ^ (r % 8).
__device__ __forceinline__ uint32_t sw128(int row, int chunk) { return (uint32_t)row * 128u + (uint32_t)((chunk ^ (row & 7)) << 4); }
__device__ __forceinline__ uint64_t tile_desc(uint32_t saddr) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)1u << 16 | (uint64_t)(1024u >> 4) << 32 | (uint64_t)1u << 46 |
         (uint64_t)2u << 61;
}
template <typename T>
__device__ constexpr uint32_t instr_desc(int n) {  // M = 128, N = n, A and B of type T, f32 result
  return (1u << 4) | (std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(0u)
      : "memory");
}
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
               : "memory");
}
// One lane of the warp.  (The compiler knows that a single lane runs what this guards: the products' operands then
// need no loop over lanes.  Guarded by a comparison of the lane's number an instruction took 95 clocks to issue.)
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_smem_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 consecutive 32-bit columns of the thread's TMEM lane (complete after tc_wait_ld / tc_wait_st).
__device__ __forceinline__ void tc_ld32(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tc_st16(uint32_t addr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tc_ld16(uint32_t addr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}

// 2^x (ex2.approx: 2 ulp; results below 2^-126 are 0)
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// pairs of f32 (one instruction for two operations)
__device__ __forceinline__ uint64_t pair2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 split2(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {  // NaN if one of them is
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float top_of(const uint32_t* x) {  // of 32 scores
  float m[2] = {__uint_as_float(x[0]), __uint_as_float(x[1])};
#pragma unroll
  for (int j = 2; j < 32; j += 2) m[j / 2 % 2] = max3(m[j / 2 % 2], __uint_as_float(x[j]), __uint_as_float(x[j + 1]));
  return max3(m[0], m[1], m[1]);
}

// The weights 2^(scale x - ref) of 32 finite (or -inf) scores, as 16 columns of P, and their sum.  The special-function
// unit makes 16 a clock, fewer than the tensor cores want: every fourth pair is computed instead, 2^y = 2^n 2^f with
// n = round(y), |f| <= 1/2 and a degree-4 polynomial for 2^f (least maximum relative error by weighted least squares:
// 2.7e-6, 0.6% of a weight's rounding to f16).  y is held at -125 from below: 2^-125 rounds to zero against a sum
// of 2^-8 or more.
template <typename T>
__device__ __forceinline__ void weigh(const uint32_t* x, uint64_t scale2, uint64_t nref2, uint64_t (&sum)[2], uint32_t at) {
  const float kMagic = 12582912.0f;  // 1.5 * 2^23: adding it rounds to an integer, in the low bits
  const uint64_t magic = pair2(kMagic, kMagic), minus = pair2(-kMagic, -kMagic), neg = pair2(-1.0f, -1.0f);
  const uint64_t c4 = pair2(0.009570102f, 0.009570102f), c3 = pair2(0.05591786f, 0.05591786f),
                 c2 = pair2(0.24024744f, 0.24024744f), c1 = pair2(0.6931218f, 0.6931218f),
                 c0 = pair2(0.9999993f, 0.9999993f);
  uint32_t p[16];
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    uint64_t y = fma2(pair2(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1])), scale2, nref2);
    float2 v = split2(y);
    float2 e;
    if (j % 4 != 3) {
      e = make_float2(ex2(v.x), ex2(v.y));
    } else {
      y = pair2(fmaxf(v.x, -125.0f), fmaxf(v.y, -125.0f));
      const uint64_t r = add2(y, magic);
      const uint64_t f = fma2(add2(r, minus), neg, y);
      uint64_t q = fma2(f, c4, c3);
      q = fma2(q, f, c2);
      q = fma2(q, f, c1);
      q = fma2(q, f, c0);
      const float2 n = split2(r), b = split2(q);
      e = make_float2(__uint_as_float(__float_as_uint(b.x) + (__float_as_uint(n.x) << 23)),
                      __uint_as_float(__float_as_uint(b.y) + (__float_as_uint(n.y) << 23)));
    }
    sum[j % 2] = add2(sum[j % 2], pair2(e.x, e.y));
    p[j] = pack2<T>(e.x, e.y);
  }
  tc_st16(at, p);
}

// 16 bytes from global to shared memory, or 16 zero bytes
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool real) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
// arrives on the barrier once the thread's copies so far have landed
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}

template <int HD>
struct Tile {
  static constexpr int kSlots = HD == 128 ? 4 : 8;         // page slots of the ring
  static constexpr uint32_t kHalf = kPageTokens * HD * 2;  // bytes of K, or V, of a page and kv head
  static constexpr uint32_t kQ = 128 * HD * 2;             // bytes of a query tile
  static constexpr int kRow = HD + kSegPad;
  // two query tiles; slots [K][V]; a staging tile of 32 x 16 floats per warp
  static constexpr uint32_t kStage = 32 * 64;
  static constexpr size_t kSmem = 2 * (size_t)kQ + (size_t)kSlots * 2 * kHalf + 8 * kStage;
};

constexpr int kSoftWarps = 4;  // softmax warps of a stream of the tile kernel
constexpr int kProducers = 32;                                  // threads of the producer warp
constexpr int kThreads = 2 * 32 * kSoftWarps + 2 * 32 + kProducers + 32;
constexpr int kFlagRing = 16;  // flags of the last pages (the producer is at most kSlots + 1 pages ahead)

// What window row i sees of its window: with ancestor sets (bits in shared memory) those, else rows 0..i.
struct Window {
  const uint32_t* anc;  // [positions][8], or null
  int positions;
  __device__ __forceinline__ bool sees(int i, int j) const {
    return j < positions && (anc ? (anc[8 * i + (j >> 5)] >> (j & 31)) & 1u : j <= i);
  }
  // bits of the 32 positions from `at` = position - base on (negative ones are committed: seen)
  __device__ __forceinline__ uint32_t word(int i, long long at) const {
    if (at <= -32) return 0xffffffffu;
    if (anc == nullptr) return at > i ? 0u : i - at >= 31 ? 0xffffffffu : (2u << (int)(i - at)) - 1u;
    if (at >= 256) return 0u;
    const int k = (int)at;
    if (k < 0) return ((1u << -k) - 1u) | anc[8 * i] << -k;
    const uint32_t lo = anc[8 * i + k / 32], hi = k / 32 < 7 ? anc[8 * i + k / 32 + 1] : 0u;
    return __funnelshift_r(lo, hi, k % 32);
  }
};

// A CTA's part of an item.
struct Segment {
  int item, kvh, x0, rows;   // item among its kind; kv head, first row, rows (<= kRowTile)
  bool group, pair;          // group entry; more than 128 rows
  int s0;                    // its (first) sequence
  int named;                 // the sequence whose table names the pages
  int page0, pages;          // table entry of the first page, pages
  int streams;               // streams with work
  __device__ __forceinline__ int stream_pages(int s) const { return pair ? pages : (pages + 1 - s) / 2; }
  __device__ __forceinline__ int stream_rows(int s) const { return pair ? (s ? rows - 128 : 128) : rows; }
};

// The CTA's segments in order: pages whose first unit lies in its share.
struct Walk {
  const Args& a;
  const Plan& plan;
  const int* first;
  uint32_t w, end;
  int e;
  __device__ __forceinline__ Walk(const Args& args, const Plan& p, const int* firsts, uint32_t begin, uint32_t finish)
      : a(args), plan(p), first(firsts), w(begin), end(finish), e(entry_at(p, args.groups.n + args.seqs.n, begin)) {}
  __device__ __forceinline__ bool next(Segment& s) {
    while (w < end) {
      while (plan.cum[e + 1] <= w) ++e;
      const Entry en = entry_of(a, e);
      const uint32_t units = units_of(en, plan.pages[e]);
      const uint32_t tile = (w - plan.cum[e]) / units, u0 = plan.cum[e] + tile * units;
      const uint32_t b0 = pages_before(en, w - u0), b1 = pages_before(en, min(units, end - u0));
      w = min(u0 + units, end);
      if (b0 >= b1) continue;
      s.item = items_before(a, e) + (int)tile;
      s.group = e < a.groups.n;
      s.s0 = en.s0;
      s.kvh = (int)tile / en.tiles;
      s.x0 = (int)tile % en.tiles * kRowTile;
      s.rows = min(en.rows - s.x0, kRowTile);
      s.pair = s.rows > 128;
      s.named = s.group ? first[e] : en.s0;
      s.page0 = (s.group ? 0 : first[e]) + (int)b0;
      s.pages = (int)(b1 - b0);
      s.streams = s.pair || s.pages > 1 ? 2 : 1;
      return true;
    }
    return false;
  }
};

// ---------------------------------------------------------------------------------------------------
// tile kernel: entries of more than 16 rows per kv head
//
// Two streams of four softmax warps each own 128 rows, one thread a row: no reductions across lanes.  With more than
// 128 rows the streams take a row tile each of every page; with fewer they take alternate pages of the same rows and
// give two partials.  A stream has two score buffers, so the scores of its next page are computed while it weighs
// this one's; its weights go back to TMEM as the first operand of their product with V.  O is rescaled only when a
// row's maximum grows by more than 2^8 (weights stay below 2^8, far inside the types' range); the first maximum of a
// segment sets the reference.
//
// Every wait is bounded.  When one gives up, all warps do: the rows whose products are missing become NaN, the caller's
// flag is raised, and the CTA ends after its products and copies in flight.
//
// A page of both streams takes 2,230 clocks, in which 16 score products (M 128, N 64, K 16, both operands in shared
// memory) complete every 107 and 8 products with V every 64, and the softmax warps are busy for about 1,900: the chain of
// scores, softmax and products bounds it, no unit alone (256 rows over 8,192 positions: tensor unit 53% of the active
// clocks, of which arithmetic 40%, special-function unit 31%, issue slots 41%).  (Score products of two pages, N 128, take
// no longer, but their scores leave no room for a second buffer: a page of both streams then waits for its own softmax,
// 3,100 clocks.  With half the query in TMEM, one score buffer: 2,750.)
//
// The producer warp copies the pages with 16-byte asynchronous copies, because the cache's chunk order is not the
// tensor cores' (128-byte swizzle): each chunk goes straight to its place, where a bulk copy would need a reordering
// pass.
// ---------------------------------------------------------------------------------------------------
template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 1) kv_tile_kernel(const __grid_constant__ Args a) {
  using TL = Tile<HD>;
  constexpr int SL = TL::kSlots;
  extern __shared__ __align__(1024) uint8_t smem[];  // [2 query tiles][slots of [K block][V block]]
  __shared__ Plan plan;
  __shared__ int s_first[kMaxEntries];
  __shared__ __align__(8) uint64_t copied_k[SL], copied_v[SL], free_k[SL], free_v[SL];
  __shared__ __align__(8) uint64_t full_k[2][SL], full_v[2][SL];  // by a stream's own count of pages
  __shared__ __align__(8) uint64_t q_ready[2], drained[2];
  // of a stream's even and odd pages (a stream is up to two pages ahead, so that one barrier's phases could be missed)
  __shared__ __align__(8) uint64_t s_full[2][2], p_ready[2][2], o_done[2][2];
  __shared__ int s_real[kFlagRing];  // the page exists
  __shared__ uint32_t s_anc[kKvMaxWindow * 8];
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_dead;  // a bounded wait gave up: the others give up too
  __shared__ volatile int s_odd;   // a value that is not finite, and that some row sees, became zero
  uint8_t* ring = smem + 2 * TL::kQ;
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  // warps: 2 x 4 softmax, then a product warp per stream, the producer and the relay
  constexpr int kMma = 2 * kSoftWarps, kProducer = kMma + 2, kRelay = kMma + 3;
  if (threadIdx.x == 0) {
    for (int s = 0; s < SL; ++s) {
      mbar_init(&copied_k[s], kProducers + 1);  // and the page flags
      mbar_init(&copied_v[s], kProducers);
      mbar_init(&free_k[s], 2);  // both streams' products (of a block that one stream uses: the same one twice)
      mbar_init(&free_v[s], 2);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_ready[s], kSoftWarps);
      for (int k = 0; k < 2; ++k) {
        mbar_init(&s_full[s][k], 1);
        mbar_init(&p_ready[s][k], kSoftWarps);
        mbar_init(&o_done[s][k], 1);
      }
      mbar_init(&drained[s], 1);
      for (int k = 0; k < SL; ++k) {
        mbar_init(&full_k[s][k], 1);
        mbar_init(&full_v[s][k], 1);
      }
    }
    mbar_fence_init();
    s_dead = (smem_addr(smem) & 1023u) != 0;  // the operand tiles' alignment
    s_odd = 0;
  }
  griddep_wait();
  griddep_launch();
  make_plan(a, &plan, s_first, 1, gridDim.x);
  if (a.parent != nullptr) make_ancestors(a, s_anc);
  publish(a, plan, 1);
  const Shares shares = plan.cut();
  if (blockIdx.x >= shares.C) return;
  if (warp == kMma) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr(&s_tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  // TMEM columns of stream s: two score buffers of 64 (a page each; its weights go over the first 32), then O at
  // 256 s + 128
  const uint32_t tmem = s_tmem;
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    const uint32_t addr = smem_addr(bar);
    for (uint32_t i = 0; i < a.polls; ++i) {
      uint32_t done;
      asm volatile(
          "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
          : "=r"(done)
          : "r"(addr), "r"(parity)
          : "memory");
      if (done) return true;
      if ((i & 255) == 255 && s_dead) return false;
    }
    s_dead = 1;
    return false;
  };
  // the same for all of a warp, whose lanes vote and elect afterwards
  auto warp_wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };

  Walk walk(a, plan, s_first, shares.begin(blockIdx.x), shares.begin(blockIdx.x + 1));
  Segment g;
  if (warp == kRelay) {
    // ---------------- relay: copies that have landed become visible to the tensor cores, for the streams that use the
    // page (the copies are generic writes; the fence would cost a product warp its time) ----------------
    if (lane == 0) {
      uint32_t idx = 0, count[2] = {0, 0};
      bool ok = true;
      while (ok && walk.next(g))
        for (int b = 0; b < g.pages && ok; ++b, ++idx) {
          const int slot = (int)(idx % SL);
          const uint32_t phase = (idx / SL) & 1u;
          const int s_begin = g.pair ? 0 : b % 2, s_end = g.pair ? 2 : s_begin + 1;
          if (!(ok = wait(&copied_k[slot], phase))) break;
          fence_smem_async();
          for (int s = s_begin; s < s_end; ++s) mbar_arrive(&full_k[s][count[s] % SL]);
          if (!(ok = wait(&copied_v[slot], phase))) break;
          fence_smem_async();
          for (int s = s_begin; s < s_end; ++s) mbar_arrive(&full_v[s][count[s]++ % SL]);
        }
    }
    __syncwarp();
  } else if (warp == kProducer) {
    // ---------------- producer: K, then V, of every page; chunks go to their swizzled places ----------------
    // K (or V) of a page is kCopies x 32 chunks of 16 bytes; the lane's i-th one is lane + 32 i.  Its place in the
    // swizzled tile repeats: a K row (of HD / 8 chunks) keeps its chunk and moves kStep rows, a V row keeps its chunk
    // and moves four rows.
    constexpr int kCopies = kPageTokens * HD / 8 / 32;
    constexpr int kStep = 32 / (HD / 8);
    const int kr = lane / (HD / 8), kc = kv_k_chunk(lane % (HD / 8), kr);  // (a stored chunk's place: its own inverse)
    const int vr = lane / 8, vc = kv_v_chunk(lane % 8, vr);
    static_assert(kStep % 2 == 0, "rows of one parity: the chunk's place repeats");
    auto k_at = [&](int i) { return (uint32_t)(kc / 8) * (kPageTokens * 128) + sw128(kr + kStep * i, kc % 8); };
    auto v_at = [&](int i) { return sw128(vr + 4 * i, vc); };
    uint32_t idx = 0;
    bool ok = true;
    while (ok && walk.next(g)) {
      const int32_t* table = a.seqs.table(g.named) + g.page0;
      // positions at or after `base` are the window's (or nobody's): values of their pages are checked
      const long long base = g.group ? 0x7fffffffffffffffll : a.seqs.base(g.s0);
      int32_t page = __ldg(table);
      for (int b = 0; b < g.pages; ++b, ++idx) {
        const int slot = (int)(idx % SL);
        const uint32_t phase = (idx / SL) & 1u;
        const bool real = page >= 0 && page < a.seqs.pool_pages;
        const size_t off = ((size_t)(real ? page : 0) * a.nkv + g.kvh) * (size_t)TL::kHalf + 16 * lane;
        if (b + 1 < g.pages) page = __ldg(table + b + 1);
        uint8_t* kd = ring + (size_t)slot * 2 * TL::kHalf;
        uint8_t* vd = kd + TL::kHalf;
        const uint32_t ka = smem_addr(kd), va = smem_addr(vd);
        if (!(ok = wait(&free_k[slot], phase ^ 1u))) break;
        if (lane == 0) {
          s_real[idx % kFlagRing] = real;
          mbar_arrive(&copied_k[slot]);
        }
        const uint8_t* src = static_cast<const uint8_t*>(a.k) + off;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) cp_async16(ka + k_at(i), src + 512 * i, real);
        cp_async_arrive(&copied_k[slot]);
        if (!(ok = wait(&free_v[slot], phase ^ 1u))) break;
        src = static_cast<const uint8_t*>(a.v) + off;
#pragma unroll
        for (int i = 0; i < kCopies; ++i) cp_async16(va + v_at(i), src + 512 * i, real);
        const long long first = (long long)(g.page0 + b) * kPageTokens;
        if (first + kPageTokens <= base) {
          cp_async_arrive(&copied_v[slot]);
        } else {
          // 0 * inf and 0 * NaN: a value that is not finite counts only for the rows that see its position.  In a
          // page with positions that some row does not see, such values become zero here, and reach the rows that see
          // them at the segment's end.
          asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 1
          for (int i = 0; i < kCopies; ++i) {
            uint4* at = reinterpret_cast<uint4*>(vd + v_at(i));
            const uint4 x = *at;
            if (!(has_nonfinite<T>(x.x) || has_nonfinite<T>(x.y) || has_nonfinite<T>(x.z) || has_nonfinite<T>(x.w))) continue;
            uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const uint32_t m = nonfinite_mask<T>(w[k / 2]) & (k & 1 ? 0xffff0000u : 0xffffu);
              const long long pos = first + 8 * vc + k;
              if (m == 0) continue;
              w[k / 2] &= ~m;
              if (pos < base + a.positions) s_odd = 1;
            }
            *at = make_uint4(w[0], w[1], w[2], w[3]);
          }
          mbar_arrive(&copied_v[slot]);
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncwarp();
  } else if (warp >= kMma) {
    // ---------------- products of stream s ----------------
    const int s = warp - kMma;
    {
      const uint32_t qa = smem_addr(smem) + s * TL::kQ, ra = smem_addr(ring), t0 = tmem + 256 * s;
      uint32_t idx0 = 0, segs = 0, done = 0, asked = 0;  // pages before the segment; the stream's segments, pages, scores
      bool ok = true;
      for (; ok && walk.next(g); idx0 += g.pages) {
        if (s >= g.streams) continue;
        const int step = g.pair ? 1 : 2;
        auto release = [&](uint64_t* bar) {  // of a page that one stream uses: for both
          tc_commit(bar);
          if (!g.pair) tc_commit(bar);
        };
        auto scores = [&](int b) {  // S = Q K^T of page b, the stream's page `asked`
          const int slot = (int)((idx0 + b) % SL);
          if (!warp_wait(&full_k[s][asked % SL], (asked / SL) & 1u)) return false;
          tc_after();
          const uint32_t k = ra + (uint32_t)slot * 2 * TL::kHalf;
          if (elect_one()) {
#pragma unroll
            for (int c = 0; c < HD / 64; ++c)
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)
                mma_ss(t0 + 64 * (asked & 1u), tile_desc(qa + c * (128 * 128) + 32 * kk),
                       tile_desc(k + c * (kPageTokens * 128) + 32 * kk), instr_desc<T>(kPageTokens), c + kk > 0);
            tc_commit(&s_full[s][asked & 1u]);
            release(&free_k[slot]);
          }
          __syncwarp();
          ++asked;
          return true;
        };
        int b = g.pair ? 0 : s;
        ok = warp_wait(&q_ready[s], segs++ & 1u) && scores(b) && (b + step >= g.pages || scores(b + step));
        for (bool first = true; ok && b < g.pages; b += step, first = false, ++done) {
          const int slot = (int)((idx0 + b) % SL);
          if (!(ok = warp_wait(&full_v[s][done % SL], (done / SL) & 1u) &&
                     warp_wait(&p_ready[s][done & 1u], (done >> 1) & 1u)))
            break;
          tc_after();
          const uint32_t v = ra + (uint32_t)slot * 2 * TL::kHalf + TL::kHalf;
          if (elect_one()) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)  // O (+)= P V
              mma_ts(t0 + 128, t0 + 64 * (done & 1u) + 8 * kk, tile_desc(v + 32 * kk), instr_desc<T>(HD), !first || kk > 0);
            tc_commit(&o_done[s][done & 1u]);
            release(&free_v[slot]);
          }
          __syncwarp();
          if (b + 2 * step < g.pages) ok = scores(b + 2 * step);  // over the weights that these products read
        }
      }
      // The accumulators are freed after the last products, also where the softmax no longer waits for them.
      if (elect_one()) tc_commit(&drained[s]);
      __syncwarp();
      mbar_wait(&drained[s], 0, nullptr);
    }
    __syncwarp();
  } else {
    // ---------------- softmax: stream s, one thread per row ----------------
    const int s = warp / kSoftWarps, r = threadIdx.x % 128;
    const Window win{a.parent ? s_anc : nullptr, a.positions};
    const uint32_t lanes = tmem + ((uint32_t)(warp % 4) * 32 << 16);
    const uint32_t ts = lanes + 256 * s, to = ts + 128;
    uint8_t* qs = smem + s * TL::kQ;
    uint8_t* stage = smem + 2 * TL::kQ + SL * 2 * TL::kHalf + warp * TL::kStage;
    uint32_t before = 0, idx0 = 0, done = 0;  // pages so far; before the segment; of the stream
    bool ok = true;
    auto advance = [&]() {  // the stream's next segment
      while (walk.next(g)) {
        idx0 = before;
        before += g.pages;
        if (s < g.streams) return true;
      }
      return false;
    };
    // the segment's rows: the thread's window row and its base, the query row to shared memory
    int nrows = 0, i = 0;
    long long base = 0;
    bool work = false, valid = false;  // the warp has a row; the thread has one
    auto load = [&]() {
      const int x = g.x0 + (g.pair ? 128 * s : 0) + r;
      nrows = g.stream_rows(s);
      work = (warp % 4) * 32 < nrows;
      valid = r < nrows;
      if (work) {
        const int srow = valid ? x / a.group : 0, head = g.kvh * a.group + (valid ? x % a.group : 0);
        const int b = g.s0 + srow / a.positions;
        i = srow % a.positions;
        base = a.seqs.base(b);
        const uint4* q = reinterpret_cast<const uint4*>(
            static_cast<const T*>(a.q) + ((long long)b * a.positions + i) * a.ld_q + (long long)head * HD);
        uint4 v[HD / 8];  // (asked for before the base is known)
#pragma unroll
        for (int c = 0; c < HD / 8; ++c) v[c] = __ldg(q + c);
        valid = valid && base >= 0;
#pragma unroll
        for (int c = 0; c < HD / 8; ++c)
          *reinterpret_cast<uint4*>(qs + (c / 8) * (128 * 128) + sw128(r, c % 8)) = valid ? v[c] : make_uint4(0u, 0u, 0u, 0u);
        fence_smem_async();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_ready[s]);
    };
    bool more = advance();
    if (more) load();
    while (more) {
      float m = -INFINITY, l = 0.0f;  // m: the reference of the weights so far (scaled scores)
      const int np = g.stream_pages(s);
      for (int t = 0; t < np; ++t, ++done) {
        ok = ok && warp_wait(&s_full[s][done & 1u], (done >> 1) & 1u);
        if (work && ok) {
          tc_after();
          const int b = g.pair ? t : 2 * t + s;
          const long long first = (long long)(g.page0 + b) * kPageTokens;
          const uint32_t tp = ts + 64 * (done & 1u);
          uint32_t x[64];
          tc_ld32(tp, x);
          tc_ld32(tp + 32, x + 32);
          const bool real = s_real[(idx0 + b) % kFlagRing];
          // whether some row of the warp does not see all of the page
          const bool masked = __any_sync(0xffffffffu, valid && (!real || first + kPageTokens > base));
          tc_wait_ld();
          if (masked)
#pragma unroll
            for (int w = 0; w < 2; ++w) {
              const uint32_t see = real ? win.word(i, first + 32 * w - base) : 0u;
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (!((see >> j) & 1u)) x[32 * w + j] = __float_as_uint(-INFINITY);
            }
          const float top = max3(top_of(x), top_of(x + 32), -INFINITY) * a.scale_log2;
          if (t == 0) {
            m = top;
          } else {
            const bool grow = top > m + 8.0f;
            if (__any_sync(0xffffffffu, grow)) {
              // the products of the page before are the last to add to O
              ok = warp_wait(&o_done[s][(done - 1) & 1u], ((done - 1) >> 1) & 1u);
              tc_after();
              const float f = grow ? ex2(m - top) : 1.0f;  // 0 for a row that had seen nothing
              if (grow) m = top;
              l *= f;
#pragma unroll 1
              for (int c = 0; c < HD / 16; ++c) {
                uint32_t o[16];
                tc_ld16(to + 16 * c, o);
                tc_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
                tc_st16(to + 16 * c, o);
              }
            }
          }
          const float ref = m == -INFINITY ? 0.0f : m;
          if (!masked && __all_sync(0xffffffffu, fabsf(top) <= FLT_MAX)) {
            const uint64_t scale2 = pair2(a.scale_log2, a.scale_log2), nref2 = pair2(-ref, -ref);
            uint64_t sum[2] = {0, 0};
            weigh<T>(x, scale2, nref2, sum, tp);
            weigh<T>(x + 32, scale2, nref2, sum, tp + 16);
            const float2 y = split2(add2(sum[0], sum[1]));
            l += y.x + y.y;
          } else {  // masked pages, and rows with infinities or NaN: the exponential itself for every score
            float sum = 0.0f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t p[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                const float p0 = ex2(fmaf(__uint_as_float(x[32 * h + 2 * j]), a.scale_log2, -ref));
                const float p1 = ex2(fmaf(__uint_as_float(x[32 * h + 2 * j + 1]), a.scale_log2, -ref));
                sum += p0 + p1;
                p[j] = pack2<T>(p0, p1);
              }
              tc_st16(tp + 16 * h, p);
            }
            l += sum;
          }
          tc_wait_st();
          tc_before();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[s][done & 1u]);
      }
      // The next segment's query rows (the scores that read this one's are complete), then this one's partial rows,
      // once its last products are complete.
      const Segment was = g;
      const int was_i = i, left = nrows - (warp % 4) * 32;
      const long long was_base = base;
      const bool was_work = work, was_valid = valid;
      if ((more = advance())) load();
      ok = ok && warp_wait(&o_done[s][(done - 1) & 1u], ((done - 1) >> 1) & 1u);
      if (was_work) {
        tc_after();
        const int seg = was.item + (int)blockIdx.x;
        const Args::Kind& kind = a.kind[was.group ? 0 : 1];
        float* rows = kind.part + ((size_t)(2 * seg + s) * kind.rows + (warp % 4) * 32) * TL::kRow;
        const bool odd = s_odd && !was.group;
#pragma unroll 1
        for (int c = 0; c < HD / 16; ++c) {
          uint32_t o[16];
          tc_ld16(to + 16 * c, o);
          tc_wait_ld();
          if (odd && was_valid)  // values that are not finite, which the row sees, in the stream's pages from the window's first
                                 // on (not another stream's: a row that sees none of this one's pages has no maximum here)
            for (int j = -(int)(was_base % kPageTokens); j < a.positions; ++j) {
              const long long pos = was_base + j, at = pos / kPageTokens - was.page0;
              if ((j >= 0 && !win.sees(was_i, j)) || at < 0 || at >= was.pages || (!was.pair && at % 2 != s)) continue;
              const int32_t page = a.seqs.table(was.s0)[pos / kPageTokens];
              if (page < 0 || page >= a.seqs.pool_pages) continue;
              const int pp = (int)(pos % kPageTokens);
#pragma unroll
              for (int d = 0; d < 16; ++d) {
                const int dim = 16 * c + d;
                const float v = to_f32(static_cast<const T*>(a.v)[(((size_t)page * a.nkv + was.kvh) * HD + dim) * kPageTokens +
                                                                  8 * kv_v_chunk(pp / 8, dim) + pp % 8]);
                if (!(fabsf(v) <= FLT_MAX)) o[d] = __float_as_uint(__uint_as_float(o[d]) + v);
              }
            }
          // through shared memory, so that four lanes write 64 bytes of a row
          auto at = [&](int row, int j) { return reinterpret_cast<uint4*>(stage + row * 64 + ((j ^ (row / 2 % 4)) << 4)); };
#pragma unroll
          for (int j = 0; j < 4; ++j) *at(lane, j) = make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int row = 8 * j + lane / 4;
            if (row < left)
              *reinterpret_cast<uint4*>(rows + (size_t)row * TL::kRow + 16 * c + 4 * (lane % 4)) = *at(row, lane % 4);
          }
          __syncwarp();
        }
        // a copy that never arrived: the rows say so
        if (lane < left) *reinterpret_cast<float2*>(rows + (size_t)lane * TL::kRow + HD) = make_float2(m, ok ? l : NAN);
        tc_before();
      }
    }
  }
  __syncthreads();
  if (threadIdx.x == 0 && s_dead && a.err != nullptr) atomicExch(a.err, kErrWaitTimeout);
  if (warp == kMma) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// ---------------------------------------------------------------------------------------------------
// stream kernel: entries of up to 16 rows per kv head
//
// A warp takes a share of the line and a row tile of 16; warps share nothing: a warp reads its operands from global
// memory in the fragments' order (every K and V chunk is used by one lane), keeps its state in registers and writes its
// own partial.  Eight warps a CTA, each with 8 to 16 KB of loads in flight, cover the memory's latency: a half page of
// head_dim 128 takes about 6,400 clocks with all warps at it, 5.7 TB/s.  The start (launch, plan, first rows and
// pages: four dependent reads) takes 8,000, which is most of a short call.
//
// Fragment mapping (mma m16n8k16, lane = 4 g + t): column n of S's n-tile jj is position 8 (n / 2) + 2 jj + n % 2 of
// the half page, so a lane's scores are positions 8 t + 2 jj + {0, 1}; the weights of n-tiles 2 kk and 2 kk + 1 are
// then the A fragment of P V's k-step kk, whose B fragment is the lane's one chunk of V (positions 8 t .. 8 t + 7).
// The dims of a score are summed in the lane's order of K chunks (any order, alike in Q and K).
// ---------------------------------------------------------------------------------------------------
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
// 16 bytes of the cache, in program order with the products
__device__ __forceinline__ uint4 load16(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
template <typename T>
constexpr uint32_t kOne = std::is_same<T, __half>::value ? 0x3C00u : 0x3F80u;

template <typename T, int HD>
__global__ void __launch_bounds__(32 * kStreamWarps, 1) kv_stream_kernel(const __grid_constant__ Args a, int second) {
  constexpr int KW = HD / 32;  // 16-byte words of a K row per lane
  constexpr int kRow = HD + kSegPad;
  // loads of the next half page before this one's products are done: head_dim 64 8 x 8,192 positions 36.1 -> 35.3 us;
  // with 128 the registers do not hold them (98.9 -> 104.8 us, 64 sequences of 2,048)
  constexpr bool kAhead = HD == 64;
  __shared__ Plan plan;
  __shared__ int s_first[kMaxEntries];
  __shared__ uint32_t s_anc[kKvMaxWindow * 8];
  __shared__ uint4 s_query[kStreamWarps][2 * KW][32];
  // After the tile kernel this one starts early: what it reads was complete before the tile kernel let it start.  The
  // combining kernel waits for this one alone, so this one waits for the tile kernel before it ends.
  if (!second) griddep_wait();
  griddep_launch();
  make_plan(a, &plan, s_first, 0, gridDim.x * kStreamWarps);
  if (a.parent != nullptr) {
    make_ancestors(a, s_anc);
    __syncthreads();
  }
  publish(a, plan, 0);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, t = lane % 4;
  const int E = a.groups.n + a.seqs.n;
  const Shares shares = plan.cut();
  // consecutive shares go to different SMs: short lines use all of them
  const uint32_t share = warp * gridDim.x + blockIdx.x;
  const Window win{a.parent ? s_anc : nullptr, a.positions};
  uint32_t w = 0, end = 0;
  int e = 0;
  if (share < shares.C) {
    w = shares.begin(share);
    end = shares.begin(share + 1);
    e = entry_at(plan, E, w);
  }
  while (w < end) {
    while (plan.cum[e + 1] <= w) ++e;
    const Entry en = entry_of(a, e);
    const uint32_t units = units_of(en, plan.pages[e]);
    const uint32_t kvh = (w - plan.cum[e]) / units, u0 = plan.cum[e] + kvh * units;
    const uint32_t off = pages_before(en, w - u0), upto = pages_before(en, min(units, end - u0));
    w = min(u0 + units, end);
    if (off >= upto) continue;
    const int halves = (int)(upto - off);
    const int half0 = (int)off % 2, first = (en.kind ? s_first[e] : 0) + (int)off / 2;
    const int32_t* table = a.seqs.table(en.kind ? en.s0 : s_first[e]) + first;
    int32_t page = 0, coming = __ldg(table);  // this page, the next entry
    // rows g and g + 8: window row and head
    int i0, i1;
    long long b0, b1;
    bool v0, v1;
    // (the warp's queries lie in shared memory: head_dim 128 has no registers left, and spills 24 bytes as it is)
    auto s_q = [&](int which, int u) { return &s_query[warp][which * KW + u][lane]; };
    auto row = [&](int which, int& i, long long& base, bool& valid) {
      const int r = g + 8 * which;
      valid = r < en.rows;
      const int srow = valid ? r / a.group : 0, head = (int)kvh * a.group + (valid ? r % a.group : 0);
      const int b = en.s0 + srow / a.positions;
      i = srow % a.positions;
      base = a.seqs.base(b);
      const uint4* p = reinterpret_cast<const uint4*>(
          static_cast<const T*>(a.q) + ((long long)b * a.positions + i) * a.ld_q + (long long)head * HD + (HD / 4) * t);
      uint4 v[KW];  // (asked for before the base is known)
#pragma unroll
      for (int u = 0; u < KW; ++u) v[u] = __ldg(p + u);
      valid = valid && base >= 0;
#pragma unroll
      for (int u = 0; u < KW; ++u) *s_q(which, u) = valid ? v[u] : make_uint4(0u, 0u, 0u, 0u);
    };
    row(0, i0, b0, v0);
    row(1, i1, b1, v1);
    float O[HD / 8][4];
#pragma unroll
    for (int n = 0; n < HD / 8; ++n) O[n][0] = O[n][1] = O[n][2] = O[n][3] = 0.0f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
    // K of the next half page (of table entry `pj`; of existing pages only) is asked for once the products with this
    // one's are made, V after the weights' products, so that loads are in flight while the warp computes.
    int pj = -1;
    const T *ks = nullptr, *vs = nullptr;
    auto advance = [&]() {  // to the next existing page, if there is one
      while (2 * ++pj < half0 + halves) {
        page = coming;
        if (2 * pj + 2 < half0 + halves) coming = __ldg(table + pj + 1);
        if (page >= 0 && page < a.seqs.pool_pages) {
          const size_t at = ((size_t)page * a.nkv + kvh) * (size_t)(kPageTokens * HD);
          ks = static_cast<const T*>(a.k) + at;
          vs = static_cast<const T*>(a.v) + at;
          return true;
        }
      }
      return false;
    };
    uint4 kw[4][KW], va[HD / 8];
    auto load_k = [&](int half) {
#pragma unroll
      for (int jj = 0; jj < 4; ++jj) {
        const int pos = 32 * half + 8 * (g / 2) + 2 * jj + (g % 2);
        const uint4* kr = reinterpret_cast<const uint4*>(ks + (size_t)pos * HD);
#pragma unroll
        for (int u = 0; u < KW; ++u) kw[jj][u] = load16(kr + kv_k_chunk(KW * t + u, pos));
      }
    };
    auto load_v = [&](int half) {
#pragma unroll
      for (int n = 0; n < HD / 8; ++n) {
        const int vrow = 8 * n + g;
        va[n] = load16(reinterpret_cast<const uint4*>(vs + (size_t)vrow * kPageTokens) + kv_v_chunk(4 * half + t, vrow));
      }
    };
    bool more = advance();
    int half = pj == 0 ? half0 : 0;
    if (kAhead && more) {
      load_k(half);
      load_v(half);
    }
#pragma unroll 1
    while (more) {
      if (!kAhead) {
        load_k(half);
        load_v(half);
      }
      const long long p_begin = (long long)(first + pj) * kPageTokens;
      {
        float S[4][4];
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) S[jj][0] = S[jj][1] = S[jj][2] = S[jj][3] = 0.0f;
#pragma unroll
        for (int u = 0; u < KW; ++u) {
          const uint4 q0 = *s_q(0, u), q1 = *s_q(1, u);
#pragma unroll
          for (int jj = 0; jj < 4; ++jj) {
            mma16<T>(S[jj], q0.x, q1.x, q0.y, q1.y, kw[jj][u].x, kw[jj][u].y);
            mma16<T>(S[jj], q0.z, q1.z, q0.w, q1.w, kw[jj][u].z, kw[jj][u].w);
          }
        }
        const bool second_half = half == 0 && 2 * pj + 1 < half0 + halves;
        more = second_half || advance();
        if (kAhead && more) load_k(second_half);
        // every position visible to every valid row of the tile
        const bool plain = __all_sync(0xffffffffu, (!v0 || p_begin + kPageTokens <= b0) && (!v1 || p_begin + kPageTokens <= b1));
        // bit x of a row's word: it sees position 8 t + x of the half page
        uint32_t see0 = v0 ? 0xffu : 0u, see1 = v1 ? 0xffu : 0u;
        if (!plain) {
          if (v0) see0 = (win.word(i0, p_begin + 32 * half - b0) >> (8 * t)) & 0xffu;
          if (v1) see1 = (win.word(i1, p_begin + 32 * half - b1) >> (8 * t)) & 0xffu;
        }
        float mx0 = m0, mx1 = m1;
#pragma unroll
        for (int jj = 0; jj < 4; ++jj)
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            S[jj][x] = (see0 >> (2 * jj + x)) & 1u ? S[jj][x] * a.scale_log2 : -INFINITY;
            S[jj][2 + x] = (see1 >> (2 * jj + x)) & 1u ? S[jj][2 + x] * a.scale_log2 : -INFINITY;
            mx0 = fmaxf(mx0, S[jj][x]);
            mx1 = fmaxf(mx1, S[jj][2 + x]);
          }
#pragma unroll
        for (int o = 1; o <= 2; o <<= 1) {
          mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, o));
          mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, o));
        }
        // a row that has seen nothing yet keeps m = -inf: its terms are 2^-inf through a zero reference
        const float r0 = mx0 == -INFINITY ? 0.0f : mx0, r1 = mx1 == -INFINITY ? 0.0f : mx1;
        if (__any_sync(0xffffffffu, mx0 > m0 || mx1 > m1)) {
          const float c0 = ex2(m0 - r0), c1 = ex2(m1 - r1);
          l0 *= c0;
          l1 *= c1;
#pragma unroll
          for (int n = 0; n < HD / 8; ++n) {
            O[n][0] *= c0;
            O[n][1] *= c0;
            O[n][2] *= c1;
            O[n][3] *= c1;
          }
        }
        m0 = mx0;
        m1 = mx1;
        uint32_t pa[4][2];
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) {
          const float p00 = ex2(S[jj][0] - r0), p01 = ex2(S[jj][1] - r0);
          const float p10 = ex2(S[jj][2] - r1), p11 = ex2(S[jj][3] - r1);
          l0 += p00 + p01;  // this lane's positions; the quad's lanes add up at the end of the segment
          l1 += p10 + p11;
          pa[jj][0] = pack2<T>(p00, p01);
          pa[jj][1] = pack2<T>(p10, p11);
        }
        if (!plain) {
          // 0 * inf and 0 * NaN: a value that is not finite counts only for the rows that see its position.  Such
          // values are replaced by zero, and a second product counts those that reach an output: infinities of each
          // sign (32 positions at most) and NaN.
          bool odd = false;
#pragma unroll
          for (int n = 0; n < HD / 8; ++n)
            odd |= has_nonfinite<T>(va[n].x) || has_nonfinite<T>(va[n].y) || has_nonfinite<T>(va[n].z) ||
                   has_nonfinite<T>(va[n].w);
          if (__any_sync(0xffffffffu, odd)) {
            uint32_t in[4][2];
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
              in[jj][0] = ((see0 >> (2 * jj)) & 1u ? kOne<T> : 0u) | ((see0 >> (2 * jj + 1)) & 1u ? kOne<T> << 16 : 0u);
              in[jj][1] = ((see1 >> (2 * jj)) & 1u ? kOne<T> : 0u) | ((see1 >> (2 * jj + 1)) & 1u ? kOne<T> << 16 : 0u);
            }
#pragma unroll
            for (int n = 0; n < HD / 8; ++n) {
              float hit[4] = {0.0f, 0.0f, 0.0f, 0.0f};
              mma16<T>(hit, in[0][0], in[0][1], in[1][0], in[1][1], nonfinite_code<T>(va[n].x), nonfinite_code<T>(va[n].y));
              mma16<T>(hit, in[2][0], in[2][1], in[3][0], in[3][1], nonfinite_code<T>(va[n].z), nonfinite_code<T>(va[n].w));
#pragma unroll
              for (int x = 0; x < 4; ++x)
                if (hit[x] > 0.0f) {
                  const int h = (int)hit[x];
                  O[n][x] += h >= 4096 || ((h & 63) && h >= 64) ? NAN : h >= 64 ? -INFINITY : INFINITY;
                }
              va[n] = make_uint4(va[n].x & ~nonfinite_mask<T>(va[n].x), va[n].y & ~nonfinite_mask<T>(va[n].y),
                                 va[n].z & ~nonfinite_mask<T>(va[n].z), va[n].w & ~nonfinite_mask<T>(va[n].w));
            }
          }
        }
#pragma unroll
        for (int n = 0; n < HD / 8; ++n) {
          mma16<T>(O[n], pa[0][0], pa[0][1], pa[1][0], pa[1][1], va[n].x, va[n].y);
          mma16<T>(O[n], pa[2][0], pa[2][1], pa[3][0], pa[3][1], va[n].z, va[n].w);
        }
        if (kAhead && more) load_v(second_half);
        half = second_half;
      }
    }
    // the segment's partial rows
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, o);
      l1 += __shfl_xor_sync(0xffffffffu, l1, o);
    }
    const Args::Kind& kind = a.kind[en.kind];
    const int seg = items_before(a, e) + (int)kvh + (int)share;
    float* dst = kind.part + ((size_t)seg * kind.rows + g) * kRow;
    if (g < en.rows) {
#pragma unroll
      for (int n = 0; n < HD / 8; ++n) *reinterpret_cast<float2*>(dst + 8 * n + 2 * t) = make_float2(O[n][0], O[n][1]);
      if (t == 0) *reinterpret_cast<float2*>(dst + HD) = make_float2(m0, l0);
    }
    if (g + 8 < en.rows) {
      dst += 8 * kRow;
#pragma unroll
      for (int n = 0; n < HD / 8; ++n) *reinterpret_cast<float2*>(dst + 8 * n + 2 * t) = make_float2(O[n][2], O[n][3]);
      if (t == 0) *reinterpret_cast<float2*>(dst + HD) = make_float2(m1, l1);
    }
  }
  if (second) griddep_wait();
}

// One warp per row and HP heads of a kv head (whose rows lie together in a segment): their partials of the group's item
// (found by lanes 0..15) and of the sequence's own (lanes 16..31, or all where it has no group), combined by their maxima.
// A lane looks up a partial and its maxima and sums; then the lanes share the outputs' columns.  Bound by the look-up's
// instructions and three dependent reads (plan; maxima, with the first partials; the others).
template <typename T, int HD, int HP>
__global__ void __launch_bounds__(256, HP == 1 ? 4 : 2) kv_combine_kernel(const __grid_constant__ Args a) {
  using TL = Tile<HD>;
  constexpr int N = HD / 32;  // outputs per lane
  constexpr int B = HP == 4 ? 2 : 4;  // partials whose loads are in flight
  const int lane = threadIdx.x % 32;
  const uint32_t id = blockIdx.x * 8 + threadIdx.x / 32, blocks = a.nh / HP;
  if (id >= (uint32_t)(a.seqs.n * a.positions) * blocks) return;
  const int head = (int)(id % blocks) * HP, row = (int)(id / blocks);
  const int b = row / a.positions, kvh = head / a.group;
  const int its_group = group_of(a, b), width = its_group < 0 ? 32 : 16;  // lanes of a kind
  const int k = lane / width + width / 32;                                // kind
  const int e = k == 0 ? its_group : a.groups.n + b;
  const Args::Kind& kind = a.kind[k];
  // the item of the rows, and the first one's place in a segment
  const Entry en = entry_of(a, e);
  const int x = (row - en.s0 * a.positions) * a.group + head % a.group;
  const int tile = kind.tile ? kvh * en.tiles + x / kRowTile : kvh;
  int r = kind.tile ? x % 128 : x;
  // in a tile of more than 128 rows a row has one partial a segment, that of its stream; else one of each stream
  const bool pair = kind.tile && min(en.rows - x / kRowTile * kRowTile, kRowTile) > 128;
  if (pair) r += x % kRowTile / 128 * kind.rows;
  const uint32_t per = kind.tile && !pair ? 2 : 1, seg_rows = kind.tile ? 2 * kind.rows : kind.rows;
  const uint32_t item = items_before(a, e) + tile;
  griddep_wait();
  griddep_launch();
  uint32_t n = 0, c0 = 0, u0 = 0, units = 0;
  Shares shares{0, 1, 0};
  if (a.seqs.base(b) >= 0) {
    units = units_of(en, kind.plan->pages[e]);
    const uint32_t cum = kind.plan->cum[e];
    shares = kind.plan->cut();
    if (units > 0) {
      u0 = cum + tile * units;
      c0 = shares.of(u0);
      n = (shares.of(u0 + units - 1) - c0 + 1) * per;
    }
  }
  const uint32_t rounds = __reduce_max_sync(0xffffffffu, (n + width - 1) / width);
  float M[HP], l[HP], acc[HP][N];
#pragma unroll
  for (int h = 0; h < HP; ++h) {
    M[h] = -INFINITY;
    l[h] = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[h][i] = 0.0f;
  }
  for (uint32_t round = 0; round < rounds; ++round) {
    const uint32_t i = width * round + lane % width;
    float2 ml[HP];
    uint32_t src = 0;  // the partials' first row
    bool have = false;
    if (i < n) {
      const uint32_t c = c0 + i / per, s = i % per;
      // pages of the item that share c holds (none, where it is narrower than a page's units; the second stream has
      // some where there are two or more)
      const uint32_t w0 = max(shares.begin(c), u0) - u0, w1 = min(units, shares.begin(c + 1) - u0);
      have = pages_before(en, w1) - pages_before(en, w0) > s;
      src = (item + c) * seg_rows + s * kind.rows + r;
    }
#pragma unroll
    for (int h = 0; h < HP; ++h)
      ml[h] = have ? *reinterpret_cast<const float2*>(kind.part + (size_t)(src + h) * TL::kRow + HD)
                   : make_float2(-INFINITY, 0.0f);
    // the first partials' loads start before the maxima are here
    uint32_t todo = __ballot_sync(0xffffffffu, have);
    float o[B][HP][N];
    int from[B];
    auto load = [&]() {
#pragma unroll
      for (int q = 0; q < B; ++q) {
        from[q] = todo ? __ffs(todo) - 1 : -1;
        const float* p = (width == 16 && from[q] < 16 ? a.kind[0].part : a.kind[1].part) +
                         (size_t)__shfl_sync(0xffffffffu, src, from[q] & 31) * TL::kRow + N * lane;
#pragma unroll
        for (int h = 0; h < HP; ++h) {
          if (todo) {
            if constexpr (N == 4) {
              const float4 v = *reinterpret_cast<const float4*>(p + h * TL::kRow);
              o[q][h][0] = v.x, o[q][h][1] = v.y, o[q][h][2] = v.z, o[q][h][3] = v.w;
            } else {
              const float2 v = *reinterpret_cast<const float2*>(p + h * TL::kRow);
              o[q][h][0] = v.x, o[q][h][1] = v.y;
            }
          } else {
#pragma unroll
            for (int j = 0; j < N; ++j) o[q][h][j] = 0.0f;
          }
        }
        todo &= todo - 1;
      }
    };
    load();
    float f[HP];
#pragma unroll
    for (int h = 0; h < HP; ++h) {
      float m = fmaxf(M[h], ml[h].x);
      for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
      const float ref = m == -INFINITY ? 0.0f : m;
      const float keep = ex2(M[h] - ref);
      f[h] = ex2(ml[h].x - ref);
      float add = ml[h].y * f[h];
      for (int d = 16; d > 0; d >>= 1) add += __shfl_xor_sync(0xffffffffu, add, d);
      M[h] = m;
      l[h] = l[h] * keep + add;
#pragma unroll
      for (int j = 0; j < N; ++j) acc[h][j] *= keep;
    }
    for (;;) {
#pragma unroll
      for (int q = 0; q < B; ++q)
#pragma unroll
        for (int h = 0; h < HP; ++h) {
          const float w = __shfl_sync(0xffffffffu, f[h], from[q] & 31);
#pragma unroll
          for (int j = 0; j < N; ++j) acc[h][j] += o[q][h][j] * (from[q] < 0 ? 0.0f : w);
        }
      if (todo == 0) break;
      load();
    }
  }
#pragma unroll
  for (int h = 0; h < HP; ++h) {
    const float inv = l[h] == 0.0f ? 0.0f : 1.0f / l[h];
    T* out = static_cast<T*>(a.out) + ((size_t)row * a.nh + head + h) * HD + N * lane;
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
      for (int i = 0; i < N; ++i) out[i] = acc[h][i] * inv;
    } else if constexpr (N == 4) {
      *reinterpret_cast<uint2*>(out) =
          make_uint2(pack2<T>(acc[h][0] * inv, acc[h][1] * inv), pack2<T>(acc[h][2] * inv, acc[h][3] * inv));
    } else {
      *reinterpret_cast<uint32_t*>(out) = pack2<T>(acc[h][0] * inv, acc[h][1] * inv);
    }
  }
}

size_t al256(size_t n) { return (n + 255) & ~(size_t)255; }

// How a call is laid out: which kernel takes the groups and which the sequences, and the workspace.
struct Layout {
  bool tile[2];     // groups, sequences: the tile kernel
  int tiles;        // row tiles of a sequence
  int rows[2];      // row capacity of a segment (tile kernel: of half of one)
  int shares[2];
  size_t items;     // of groups and sequences
  size_t plan, part[2];  // bytes
  size_t total() const { return 2 * plan + part[0] + part[1]; }
};

Layout layout_of(int n, int positions, int nh, int nkv, int hd, const KvGroups& groups, int sm_count) {
  Layout s;
  const int rows = positions * (nh / nkv);
  int most = 0;  // rows of the largest group
  bool any = false;
  for (int g = 0; g < groups.n; ++g)
    if (groups.pages[g] > 0) {
      any = true;
      most = std::max(most, (groups.start[g + 1] - groups.start[g]) * rows);
    }
  const int widest[2] = {most, rows};
  s.tile[1] = rows > kStreamRows;
  s.tile[0] = any ? most > kStreamRows : s.tile[1];  // without shared pages there is one kernel
  s.tiles = s.tile[1] ? (rows + kRowTile - 1) / kRowTile : 1;
  size_t items[2] = {0, (size_t)n * s.tiles * nkv};
  for (int g = 0; g < groups.n; ++g)
    items[0] += (s.tile[0] ? (size_t)((groups.start[g + 1] - groups.start[g]) * rows + kRowTile - 1) / kRowTile : 1) * nkv;
  s.items = items[0] + items[1];
  s.plan = al256(sizeof(Plan));
  for (int k = 0; k < 2; ++k) {
    s.rows[k] = s.tile[k] ? std::min(k ? rows : 128, 128) : std::max(1, widest[k]);
    s.shares[k] = s.tile[k] ? sm_count : sm_count * kStreamWarps;
    s.part[k] = k == 0 && !any ? 0
                               : al256((items[k] + s.shares[k]) * (s.tile[k] ? 2 : 1) * s.rows[k] * (size_t)(hd + kSegPad) *
                                       sizeof(float));
  }
  return s;
}

template <typename T, typename O, int HD>
int launch_typed(const Args& a, const Layout& s, int sm_count, cudaStream_t st) {
  using TL = Tile<HD>;
  const bool tiled = s.tile[0] || s.tile[1];
  if (tiled) {
    CLM_TRY(ensure_smem(kv_tile_kernel<T, HD>, TL::kSmem));
    CLM_TRY(launch_pdl(kv_tile_kernel<T, HD>, dim3((unsigned)sm_count), dim3(kThreads), TL::kSmem, st, a));
  }
  // (on the default streams launches do not overlap, and the second one need not wait)
  if (!s.tile[0] || !s.tile[1])
    CLM_TRY(launch_pdl(kv_stream_kernel<T, HD>, dim3((unsigned)sm_count), dim3(32 * kStreamWarps), 0, st, a, (int)tiled));
  const uint64_t rows = (uint64_t)a.seqs.n * a.positions * a.nh;
  auto combine = [&](auto kernel, int heads) {
    return launch_pdl(kernel, dim3((unsigned)ceil_div(rows / heads, 8)), dim3(256), 0, st, a);
  };
  // Several heads a warp where one each would be more than the GPU holds at once: the look-up is done once for them (8,192
  // rows and heads of 128 with six partials each: 13 -> 9 us; but 1,024 of 64 with twenty: 10 -> 16).
  const bool many = rows > 32ull * sm_count;
  if (many && a.group % 4 == 0) return combine(kv_combine_kernel<O, HD, 4>, 4);
  if (many && a.group % 2 == 0) return combine(kv_combine_kernel<O, HD, 2>, 2);
  return combine(kv_combine_kernel<O, HD, 1>, 1);
}

}  // namespace

size_t kv_attention_work(int n, int positions, int nh, int nkv, int hd, const KvGroups& groups, int sm_count) {
  return layout_of(n, positions, nh, nkv, hd, groups, sm_count).total();
}

int launch_kv_attention(const KvAttnArgs& in, cudaStream_t st) {
  const Layout s = layout_of(in.seqs.n, in.positions, in.nh, in.nkv, in.hd, in.groups, in.sm_count);
  CLM_CHECK(s.items * (size_t)(in.seqs.max_pages + kSwitch) < (1ull << 31), CLM_OUT_OF_RANGE,
            "attention: too many pages in one call (narrower page tables, or fewer sequences)");
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
  // (a zero scale weighs all positions alike: a product with a masked score of -inf must not become NaN)
  a.scale_log2 = std::max(in.scale * 1.4426950408889634f, FLT_MIN);
  a.polls = in.polls;
  a.err = in.err;
  uint8_t* w = static_cast<uint8_t*>(in.work);
  for (int k = 0; k < 2; ++k) {
    a.kind[k].plan = reinterpret_cast<Plan*>(w + (s.tile[k] ? 0 : s.plan));  // one plan per kernel
    a.kind[k].part = reinterpret_cast<float*>(w + 2 * s.plan + (k ? s.part[0] : 0));
    a.kind[k].rows = s.rows[k];
    a.kind[k].tiles = s.tiles;
    a.kind[k].tile = s.tile[k];
  }
  const bool h = in.type == CLM_DTYPE_F16, f32 = in.out_type == CLM_DTYPE_F32;
  if (in.hd == 64) {
    if (h) return f32 ? launch_typed<__half, float, 64>(a, s, in.sm_count, st) : launch_typed<__half, __half, 64>(a, s, in.sm_count, st);
    return f32 ? launch_typed<__nv_bfloat16, float, 64>(a, s, in.sm_count, st)
               : launch_typed<__nv_bfloat16, __nv_bfloat16, 64>(a, s, in.sm_count, st);
  }
  CLM_CHECK(in.hd == 128, CLM_UNIMPLEMENTED, "head_dim 64 or 128");
  if (h) return f32 ? launch_typed<__half, float, 128>(a, s, in.sm_count, st) : launch_typed<__half, __half, 128>(a, s, in.sm_count, st);
  return f32 ? launch_typed<__nv_bfloat16, float, 128>(a, s, in.sm_count, st)
             : launch_typed<__nv_bfloat16, __nv_bfloat16, 128>(a, s, in.sm_count, st);
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
  CLM_CHECK(scale >= 0.0f && scale <= 1e30f, CLM_INVALID_ARGUMENT, "the scale must be a number that is not negative");
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
  a.polls = ctx->attention_polls;
  CLM_SCOPE(ctx);
  return launch_kv_attention(a, pick_stream(ctx, stream));
}

int clm_b200_kv_attention_wait_limit(clm_b200_ctx* ctx, uint32_t polls) {
  CLM_CHECK(ctx != nullptr, CLM_INVALID_ARGUMENT, "null context");
  ctx->attention_polls = polls;
  return CLM_OK;
}

}  // extern "C"
