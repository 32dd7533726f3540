// sample_logits.cu — temperature, top-k, top-p and min-p sampling straight from logits, one launch, no scratch.
//
// Row: d_i = l_i - max l (f32, as distribution() forms it), e_i = exp(d_i / T).  In the order (d descending, index
// ascending) three prefixes are allowed: the first top_k entries; the shortest prefix whose mass reaches top_p of the
// whole row's; the entries with e_i >= min_p.  The token is the first allowed index i, in index order, with
// u W < sum of e_j over allowed j <= i (W: the allowed mass), as sample_from walks a distribution.
//
// Masses are integers: w_i = round(2^44 e_i), evaluated with a relative error below 1e-12, summed in 64 bits.  Sums of
// integers do not depend on their order, so a row's result is the same whatever computed it, every comparison is
// exact on the w_i, and an entry below 2^-45 of the largest has no mass.
//
// A cluster of eight CTAs (sixteen for few rows) holds a row in shared memory, a slice each, so the logits are read from
// memory once however many passes the row needs:
//   1. load, maximum (and its lowest index: greedy rows end here);
//   2. without top-k / top-p: the masses of the CTAs' warp segments;
//      with them: the row's whole mass and a histogram of the entries over 64 bins per octave of e, whose counts bound
//      the cumulative mass within 1.1%: the cut falls into known bins.  Entries above these are allowed (their exact
//      mass is summed), entries below are not, and the few in them are ranked: their key range in 64 parts with exact
//      masses, then the members of the cut's part one against the other.  Where kCand or more entries share those
//      bins (a flat row, or equal logits, as from 16-bit types), their key range is divided again; where one key value
//      is left, its lowest indices stay.
//   3. the cumulative mass over CTAs, then warp segments, then entries locates the token.
//
// One row of 128,256 takes 15 us on sixteen CTAs (on eight 16 us, 27,000 clocks, of which eight barriers and what waits for
// them take half).  64 of 151,936 with top-p take 69 us: two rows' slices on an SM at a time, two waves of 52,000 clocks
// with half the issue slots used; ranking and the histogram's merging and scanning, which all CTAs of a row do alike, take
// twice as long as the first pass over the entries, and two CTAs an SM leave 64 registers a thread, with 168 bytes
// spilled.  256 of 128,256 with mixed settings take 158 us.
#include <cooperative_groups.h>

#include <cfloat>

#include "kv_ops.cuh"
#include "pdl.cuh"

namespace clm {

namespace {

namespace cg = cooperative_groups;

constexpr int kCl = 8, kWide = 16;  // CTAs of a row; of few rows
constexpr int kThr = 512;
constexpr int kWrp = kThr / 32;    // warp segments of a CTA's slice
constexpr int kBinsOct = 64;       // histogram bins per octave
constexpr int kBins = 44 * kBinsOct;
constexpr int kCand = 1024;        // candidates of a row that are ranked are fewer
constexpr int kMine = 384;         // of one CTA
constexpr int kSub = 64;           // parts of the candidates' key range
constexpr int kFrac = 44;          // fraction bits of a mass
constexpr uint32_t kMaxVocab = 8 * 48128;  // a slice and the tables fit in 227 KB

typedef unsigned long long u64;

struct Cand {
  uint32_t u, idx;  // |d| (ascends as the order does) and index
  u64 w;
};

// A sum of fewer than 1,024 masses (of up to 2^44 each), by two 32-bit atomic additions: shared memory has them in
// hardware, where a 64-bit one is a loop.
struct Split {
  uint32_t hi, lo;
  __device__ __forceinline__ void add(u64 w) {
    atomicAdd(&hi, (uint32_t)(w >> 22));
    atomicAdd(&lo, (uint32_t)w & 0x3fffffu);
  }
  __device__ __forceinline__ u64 sum() const { return ((u64)hi << 22) + lo; }
};

struct SampleArgs {
  const void* logits;
  long long ld;
  uint32_t V, slice;
  const float *temp, *top_p, *min_p;
  const int32_t* top_k;
  const double* u;
  int32_t* token;
  float* prob;
  int vec;  // rows and slices start 16-byte aligned
};

// round(2^44 * 2^y) for -48 < y <= 0: 2^y = 2^n 2^(j / 64) 2^f with |f| <= 1/128, a table of the 2^(j / 64) and a
// degree-3 polynomial for 2^f (least maximum relative error by weighted least squares: 4.5e-12).  Eight double
// operations; a polynomial alone takes thirteen and measured 12% slower in the passes that evaluate every entry.
// n64: 64 y rounded to an integer.
__device__ __forceinline__ u64 mass_of(double y, const double* table, int& n64) {
  constexpr double kShift = 0x1.8p52, kShift64 = 0x1.8p46;
  const double k = y + kShift64;
  const int n = n64 = (int)(unsigned)__double_as_longlong(k);
  const double f = y - (k - kShift64);
  double p = 0x1.c6b0616cd9777p-5;
  p = fma(p, f, 0x1.ebfc2ec2e07ffp-3);
  p = fma(p, f, 0x1.62e42fefb2b20p-1);
  p = fma(p, f, 0x1.fffffffff626bp-1);
  const double t = table[n & 63];
  const double scale = __hiloint2double(__double2hiint(t) + (((n >> 6) + kFrac) << 20), __double2loint(t));
  return (u64)(__double_as_longlong(fma(p, scale, kShift)) - __double_as_longlong(kShift));
}

// Order of floats as integers (ascending).
__device__ __forceinline__ uint32_t ord_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_ord(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }

__device__ __forceinline__ u64 warp_sum(u64 x) {
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

template <int CL>  // CTAs of a row
struct Shared {
  u64 top[CL];       // (ordered maximum, ~index) of each CTA's slice
  u64 total[CL];     // whole mass (pass 2)
  u64 above[CL];     // mass above the candidates
  u64 kept[CL];      // allowed mass
  uint32_t ncand[CL], umin[CL], umax[CL];  // candidates: how many, their key range
  uint32_t ties[CL];
  u64 half_mass[CL];       // of the lower half of the keys that are left, where a level halves them: slots that look()
  uint32_t half_count[CL];  // does not write, so that its barriers lie between two uses of them
  u64 seg[kWrp];      // allowed mass of the warp segments
  u64 red[kWrp];
  uint32_t redc[kWrp];
  float redf[2][kWrp];
  uint32_t sub_cnt[kSub];
  Split sub_mass[kSub], seg_add[kWrp];
  uint32_t cand_n, cut_n;
  double table[64];     // 2^(j / 64)
  int lo, hi;
  uint32_t cnt_before;
};

// Sums over the CTA of one value per warp (slots of shared memory; every thread gets the sum).
__device__ __forceinline__ u64 cta_sum(u64 warp_value, u64* slots, int warp, int lane) {
  __syncthreads();
  if (lane == 0) slots[warp] = warp_value;
  __syncthreads();
  return warp_sum(lane < kWrp ? slots[lane] : 0ull);
}
__device__ __forceinline__ uint32_t cta_sum(uint32_t warp_value, uint32_t* slots, int warp, int lane) {
  __syncthreads();
  if (lane == 0) slots[warp] = warp_value;
  __syncthreads();
  return __reduce_add_sync(0xffffffffu, lane < kWrp ? slots[lane] : 0u);
}

template <typename S, int CL>
__global__ void __cluster_dims__(CL, 1, 1) __launch_bounds__(kThr, CL == kCl ? 2 : 1)
    sample_logits_kernel(const __grid_constant__ SampleArgs a) {
  extern __shared__ __align__(16) uint8_t sl_smem[];
  __shared__ Shared<CL> s;
  cg::cluster_group cluster = cg::this_cluster();
  float* key = reinterpret_cast<float*>(sl_smem);  // [slice], padded with -inf
  uint32_t* hist = reinterpret_cast<uint32_t*>(key + a.slice);
  uint32_t* tot = hist + kBins;  // the row's histogram
  // once the histograms are read, their memory holds the row's candidates and this CTA's
  Cand* all = reinterpret_cast<Cand*>(hist);
  Cand* mine = all + kCand;
  static_assert(sizeof(Cand) * (kCand + kMine) <= 2 * kBins * sizeof(uint32_t), "the candidates fit over the histograms");
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const uint32_t rank = cluster.block_rank(), row = blockIdx.x / CL;
  const uint32_t v0 = min(a.V, rank * a.slice), cnt = min(a.V, v0 + a.slice) - v0;
  // a value of this CTA goes to every CTA of the row
  auto push = [&](auto* slot, auto value) {
    if (tid < CL) *cluster.map_shared_rank(slot + rank, tid) = value;
  };
  for (int i = tid; i < kBins; i += kThr) hist[i] = 0;
  if (tid < 64) s.table[tid] = exp2(tid / 64.0);
  cluster.barrier_arrive();  // waited for before the first write into another CTA's shared memory
  griddep_wait();
  griddep_launch();

  const float T = a.temp ? a.temp[row] : 1.0f;
  const int32_t k_in = a.top_k ? a.top_k[row] : 0;
  const float p_in = a.top_p ? a.top_p[row] : 1.0f, m_in = a.min_p ? a.min_p[row] : 0.0f;

  // ---- 1. load and maximum (NaN counts as -inf; -0 as 0)
  const S* src = static_cast<const S*>(a.logits) + (long long)row * a.ld + v0;
  float mx = -INFINITY;
  auto clean = [&](float x) {
    x = x == x ? x + 0.0f : -INFINITY;
    mx = fmaxf(mx, x);
    return x;
  };
  if (a.vec) {
    constexpr int N = 16 / sizeof(S);
    const uint32_t nv = cnt / N;
#pragma unroll 4
    for (uint32_t i = tid; i < nv; i += kThr) {
      const uint4 w = __ldcs(reinterpret_cast<const uint4*>(src) + i);
      S e[N];
      memcpy(e, &w, 16);
#pragma unroll
      for (int j = 0; j < N; j += 4)
        *reinterpret_cast<float4*>(key + i * N + j) =
            make_float4(clean(to_f32(e[j])), clean(to_f32(e[j + 1])), clean(to_f32(e[j + 2])), clean(to_f32(e[j + 3])));
    }
    for (uint32_t i = nv * N + tid; i < cnt; i += kThr) key[i] = clean(to_f32(src[i]));
  } else {
#pragma unroll 4
    for (uint32_t i = tid; i < cnt; i += kThr) key[i] = clean(to_f32(src[i]));
  }
  for (uint32_t i = cnt + tid; i < a.slice; i += kThr) key[i] = -INFINITY;
  const bool greedy = !(T > 0.0f);
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if (lane == 0) s.redf[0][warp] = mx;
  __syncthreads();
  mx = s.redf[0][lane % kWrp];
  for (int o = kWrp / 2; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  uint32_t first = 0xffffffffu;  // lowest index of the slice's maximum (greedy rows)
  if (greedy) {
    for (uint32_t i = tid; i < cnt; i += kThr)
      if (key[i] == mx) first = min(first, v0 + i);
    first = __reduce_min_sync(0xffffffffu, first);
    if (lane == 0) s.redc[warp] = first;
    __syncthreads();
    first = __reduce_min_sync(0xffffffffu, s.redc[lane % kWrp]);
  }
  cluster.barrier_wait();  // every CTA of the row runs
  push(s.top, (u64)ord_of(mx) << 32 | (u64)(0xffffffffu - first));
  cluster.barrier_arrive();
  // (the row's settings, while the maxima arrive)
  const double c = 1.4426950408889634 / (double)T;  // y = c d: e = 2^y
  const bool need_k = k_in > 0 && (uint32_t)k_in < a.V, need_p = p_in < 1.0f;
  const uint32_t k = need_k ? (uint32_t)k_in : 0xffffffffu;
  // entries below dcut have no mass (y < -45: it rounds to zero); entries below dlow are not allowed: dcut, or the
  // first float whose y is log2(min_p) or more
  const float dcut = fmaxf(-FLT_MAX, (float)(-45.5 / c));
  float dlow = dcut;
  if (m_in > 0.0f && !greedy) {
    const double ymin = log2((double)fminf(m_in, 1.0f));
    float d = fminf(0.0f, fmaxf(-FLT_MAX, (float)(ymin / c)));
    while (d < 0.0f && (double)d * c < ymin) d = nextafterf(d, 0.0f);
    while (d > -FLT_MAX && (double)nextafterf(d, -INFINITY) * c >= ymin) d = nextafterf(d, -INFINITY);
    dlow = fmaxf(dcut, d);
  }
  cluster.barrier_wait();
  u64 best = 0;
#pragma unroll
  for (int r = 0; r < CL; ++r) best = max(best, s.top[r]);
  const float M = of_ord((uint32_t)(best >> 32));
  if (greedy || M == -INFINITY) {  // the same for the whole cluster
    if (rank == 0 && tid == 0) {
      a.token[row] = M == -INFINITY ? -1 : (int32_t)(0xffffffffu - (uint32_t)best);
      if (a.prob) a.prob[row] = M == -INFINITY ? 0.0f : 1.0f;
    }
    return;
  }

  // ---- 2. what is allowed
  float top = M;
  if (M == INFINITY) {  // the infinite entries share the whole mass
    __syncthreads();
    for (uint32_t i = tid; i < a.slice; i += kThr) key[i] = key[i] == M ? 0.0f : -INFINITY;
    top = 0.0f;
    __syncthreads();
  }
  auto d_of = [&](float x) { return __fsub_rn(x, top); };
  auto mass_n = [&](float d, int& n) { return mass_of((double)fmaxf(d, dcut) * c, s.table, n); };  // of d >= dcut
  auto mass = [&](float d) {
    int n;
    return mass_n(d, n);
  };
  auto u_of = [&](float d) { return __float_as_uint(fabsf(d)); };  // ascends as the order does
  const uint32_t seg = (a.slice / 4 + kWrp - 1) / kWrp * 4;
  const uint32_t s0 = min(a.slice, warp * seg), s1 = min(a.slice, s0 + seg);  // this warp's segment
  // f(index, d) for the segment's entries, four consecutive ones a lane at a time (independent chains)
  auto each = [&](auto&& f) {
    for (uint32_t i = s0 + 4 * lane; i < s1; i += 128) {
      const float4 x = *reinterpret_cast<const float4*>(key + i);
      f(i, d_of(x.x));
      f(i + 1, d_of(x.y));
      f(i + 2, d_of(x.z));
      f(i + 3, d_of(x.w));
    }
  };
  // allowed entries: d >= dlow, u <= umax, key not struck out
  uint32_t umax = 0x7f7fffffu;
  u64 seg_mass = 0;
  if (!need_k && !need_p) {
    each([&](uint32_t, float d) { seg_mass += d >= dlow ? mass(d) : 0ull; });
    seg_mass = warp_sum(seg_mass);
  } else {
    // The cut is located level by level.  A level looks at the entries with keys in [ul, uh]: those before are allowed
    // (cnt_above of them, with the mass `above`), those behind are not.  Level 0 has all entries in bins of 1/64
    // octave of e; the others divide what is left evenly.
    uint32_t ul = 0, uh = umax, span = umax, cand = 0, before = 0, cnt_above = 0, most = 0;
    uint32_t in[CL];  // candidates of each CTA
    u64 above = 0, thr = ~0ull;
    bool struck = false;
    auto look = [&](auto level0) {  // (two copies of the code: level 0 reads every entry)
      constexpr bool kFirst = decltype(level0)::value;
      const float inv = (float)kBins / ((float)(uh - ul) + 1.0f);
      auto bin_of = [&](float d) {  // ascends as the order does
        if (!kFirst) return min(kBins - 1, (int)((float)(u_of(d) - ul) * inv));
        int n;
        mass_n(d, n);
        return min(kBins - 1, -n);
      };
      auto inside = [&](float d) { return d >= dlow && (kFirst || (u_of(d) >= ul && u_of(d) <= uh)); };
      u64 sum = 0;
      if (kFirst && need_p) {
        each([&](uint32_t, float d) {
          int n;
          const u64 w = mass_n(d, n);
          if (d >= dcut) sum += w;
          if (d >= dlow) atomicAdd(&hist[min(kBins - 1, -n)], 1u);
        });
      } else {
        each([&](uint32_t, float d) {
          if (inside(d)) atomicAdd(&hist[bin_of(d)], 1u);
        });
      }
      push(s.total, cta_sum(warp_sum(sum), s.red, warp, lane));
      cluster.sync();
      for (int b = tid; b < (kBins / CL); b += kThr) {
        const int bin = (int)rank * (kBins / CL) + b;
        uint32_t part[CL], n = 0;
#pragma unroll
        for (int r = 0; r < CL; ++r) part[r] = cluster.map_shared_rank(hist, r)[bin];
#pragma unroll
        for (int r = 0; r < CL; ++r) n += part[r];
#pragma unroll
        for (int r = 0; r < CL; ++r) cluster.map_shared_rank(tot, r)[bin] = n;
      }
      if (tid == 0) {
        s.lo = kBins;
        s.hi = kBins;
        s.cand_n = 0;
      }
      cluster.sync();
      if (kFirst && need_p) {
        // allowed by top-p: entries with less than `thr` mass before them (p in units of 2^-40, rounded up)
        u64 total = 0;
#pragma unroll
        for (int r = 0; r < CL; ++r) total += s.total[r];
        const u64 pi = (u64)ceil(fmax((double)p_in, 0.0) * 0x1p40);
        const u64 ph = __umul64hi(pi, total), pl = pi * total;
        thr = (ph << 24 | pl >> 40) + ((pl & 0xffffffffffull) != 0);
        if (thr == 0) thr = 1;
      }
      // cumulative counts, and masses were every entry at its bin's upper (lower) edge; 1e-4 covers the roundings of
      // the edges and of these f32 sums, which only bound where the cut can be
      constexpr int kPer = (kBins + kThr - 1) / kThr;
      auto edge = [&](int bin) {  // e at a bin's upper edge, in units of 2^-44
        if (kFirst) return exp2f((float)kFrac - ((float)bin - 0.5f) * (1.0f / kBinsOct));
        const float step = ((float)(uh - ul) + 1.0f) * (1.0f / kBins);
        // (in double: a tiny temperature's c is no float)
        return exp2f((float)(kFrac - (double)__uint_as_float(min(uh, ul + (uint32_t)((float)bin * step) + (bin > 0))) * c));
      };
      uint32_t n[kPer];
      float up[kPer], down[kPer];
      uint32_t nsum = 0;
      float usum = 0.0f, dsum = 0.0f;
      float begin = edge(tid * kPer);
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int bin = tid * kPer + j;
        const float next = edge(bin + 1);
        n[j] = bin < kBins ? tot[bin] : 0u;
        up[j] = n[j] ? (float)n[j] * begin * 1.0001f : 0.0f;
        down[j] = n[j] ? (float)n[j] * next * 0.9999f : 0.0f;
        begin = next;
        nsum += n[j];
        usum += up[j];
        dsum += down[j];
      }
      uint32_t nx = nsum;
      float ux = usum, dx = dsum;
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t on = __shfl_up_sync(0xffffffffu, nx, o);
        const float ou = __shfl_up_sync(0xffffffffu, ux, o), od = __shfl_up_sync(0xffffffffu, dx, o);
        if (lane >= o) {
          nx += on;
          ux += ou;
          dx += od;
        }
      }
      if (lane == 31) {
        s.redc[warp] = nx;
        s.redf[0][warp] = ux;
        s.redf[1][warp] = dx;
      }
      __syncthreads();
      {
        nx += __reduce_add_sync(0xffffffffu, lane < warp ? s.redc[lane % kWrp] : 0u) - nsum;
        float bu = lane < warp ? s.redf[0][lane % kWrp] : 0.0f, bd = lane < warp ? s.redf[1][lane % kWrp] : 0.0f;
        for (int o = kWrp / 2; o > 0; o >>= 1) {
          bu += __shfl_xor_sync(0xffffffffu, bu, o);
          bd += __shfl_xor_sync(0xffffffffu, bd, o);
        }
        ux += __shfl_sync(0xffffffffu, bu, 0) - usum;
        dx += __shfl_sync(0xffffffffu, bd, 0) - dsum;
      }
      const float need = (float)(thr - above);
      int lo_mine = kBins, hi_mine = kBins;
      uint32_t before_lo = 0;
#pragma unroll
      for (int j = 0; j < kPer; ++j) {
        const int bin = tid * kPer + j;
        const uint32_t n0 = nx;
        nx += n[j];
        ux += up[j];
        dx += down[j];
        const bool by_k = n[j] && nx >= k - cnt_above;
        if (lo_mine == kBins && (by_k || (n[j] && need_p && ux >= need))) {
          lo_mine = bin;
          before_lo = n0;
        }
        if (hi_mine == kBins && (by_k || (n[j] && need_p && dx >= need))) hi_mine = bin;
      }
      if (lo_mine < kBins) atomicMin(&s.lo, lo_mine);
      if (hi_mine < kBins) atomicMin(&s.hi, hi_mine);
      __syncthreads();
      const int lo = s.lo, hi = s.hi;
      if (lo_mine == lo && lo < kBins) s.cnt_before = before_lo;  // (one thread)
      // Bins ascend with u: the first u of a bin or a later one, so that the entries need no bins again.  Of level 0 it lies
      // at the bin's edge but for a few units, which the lanes try; else (and for bins past the last one) by a search of
      // 32 parts a step.  (The same in every warp.)
      auto first_of = [&](int bin) -> uint32_t {
        if (kFirst && bin < kBins) {
          if (bin <= 0) return ul;
          const uint32_t from = max(__float_as_uint((float)(((double)bin - 0.5) / (kBinsOct * c))), 16u) - 16u;
          const uint32_t under = __ballot_sync(0xffffffffu, bin_of(-__uint_as_float(from + lane)) < bin);
          if ((under & 1u) && !(under >> 31)) return from + __popc(under);
        }
        uint32_t at = ul, left = uh - ul + 1;  // the first is in [at, at + left]
        while (left > 0) {
          const uint32_t step = (left + 31) / 32, probe = at + min(left, (lane + 1) * step) - 1;
          const uint32_t under = __popc(__ballot_sync(0xffffffffu, bin_of(-__uint_as_float(probe)) < bin));
          const uint32_t skip = min(left, under * step);
          at += skip;
          left = under == 32 ? 0 : min(left - skip, step - 1);
        }
        return at;
      };
      const uint32_t ulo = first_of(lo), uhi = lo == kBins ? ulo : first_of(hi + 1);
      const float dtop = -__uint_as_float(ul);
      // before the cut's bins: dtop >= d > dlo (and d >= dlow); in them: dlo >= d >= dhi
      const float dlo = -__uint_as_float(ulo), dhi = uhi > ul ? fmaxf(dlow, -__uint_as_float(uhi - 1)) : INFINITY;
      // the masses of entries before the cut's bins and the
      // candidates
      uint32_t least = 0xffffffffu, largest = 0;
      // first which entries of up to 2,048 (a bit for each of a lane's 64), then one after the other: lanes have unlike
      // numbers of them, which even out over many
      for (uint32_t c0 = s0; c0 < s1; c0 += 2048) {
        u64 counts = 0;
        const uint32_t c1 = min(s1, c0 + 2048);
#pragma unroll 1
        for (uint32_t k = 0; c0 + 256 * k < c1; ++k) {
          const uint32_t i = c0 + 256 * k + 4 * lane;
          float x[8];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float4 v = i + 128 * h < c1 ? *reinterpret_cast<const float4*>(key + i + 128 * h)
                                              : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            x[4 * h] = v.x, x[4 * h + 1] = v.y, x[4 * h + 2] = v.z, x[4 * h + 3] = v.w;
          }
          if (d_of(fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])))) < dhi)
            continue;
          uint32_t bits = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (d_of(x[j]) >= dhi && (kFirst || d_of(x[j]) <= dtop)) bits |= 1u << j;
          counts |= (u64)bits << (8 * k);
        }
        for (; counts; counts &= counts - 1) {
          const int j = __ffsll((long long)counts) - 1;
          const uint32_t e = c0 + 128 * (j / 4) + 4 * lane + j % 4;
          const float d = d_of(key[e]);
          if (d > dlo) {
            seg_mass += mass(d);
          } else {
            const uint32_t u = u_of(d), at = atomicAdd(&s.cand_n, 1u);
            least = min(least, u);
            largest = max(largest, u);
            // (in the place of the histograms, which every CTA has read; its mass follows)
            if (at < kMine) mine[at] = Cand{u, v0 + e, 0ull};
          }
        }
      }
      const u64 level_mass = warp_sum(seg_mass);  // with the levels before
      const u64 x = cta_sum(level_mass, s.seg, warp, lane);
      for (uint32_t i = tid; i < min(s.cand_n, (uint32_t)kMine); i += kThr) mine[i].w = mass(-__uint_as_float(mine[i].u));
      push(s.above, x);
      push(s.ncand, s.cand_n);
      least = __reduce_min_sync(0xffffffffu, least);
      largest = __reduce_max_sync(0xffffffffu, largest);
      if (lane == 0) {
        s.redc[warp] = least;
        s.redf[0][warp] = __uint_as_float(largest);
      }
      __syncthreads();
      push(s.umin, __reduce_min_sync(0xffffffffu, s.redc[lane % kWrp]));
      push(s.umax, __reduce_max_sync(0xffffffffu, __float_as_uint(s.redf[0][lane % kWrp])));
      if (lo < kBins) cnt_above += s.cnt_before;
      cluster.sync();
      above = 0;
      cand = before = most = 0;
      uint32_t nl = 0xffffffffu, nh = 0;
#pragma unroll
      for (int r = 0; r < CL; ++r) {
        above += s.above[r];
        in[r] = s.ncand[r];
        if (r < (int)rank) before += in[r];
        cand += in[r];
        most = max(most, in[r]);
        nl = min(nl, s.umin[r]);
        nh = max(nh, s.umax[r]);
      }
      const bool all_allowed = lo == kBins;
      if (!all_allowed) {
        ul = nl;
        uh = umax = nh;
      }
      return all_allowed || (cand < kCand && most <= kMine);
    };
    bool done = look(std::true_type{});
    for (int level = 1; !done; ++level) {
      if (ul == uh) {
        // one key value: its `stay` lowest indices are allowed
        struck = true;
        const u64 w = mass(-__uint_as_float(ul));
        u64 stay = ~0ull;
        if (need_k) stay = k - cnt_above;
        if (need_p && w > 0) stay = min(stay, (thr - above + w - 1) / w);
        uint32_t ties = 0;
        for (uint32_t i0 = s0; i0 < s1; i0 += 32) {
          const uint32_t i = i0 + lane;
          ties += __popc(__ballot_sync(0xffffffffu, i < s1 && u_of(d_of(key[i])) == ul));
        }
        const uint32_t all_ties = cta_sum(ties, s.redc, warp, lane);
        const uint32_t first_rank = __reduce_add_sync(0xffffffffu, lane < warp ? s.redc[lane % kWrp] : 0u);
        push(s.ties, all_ties);
        cluster.sync();
        u64 rank_in = first_rank;
        for (int r = 0; r < (int)rank; ++r) rank_in += s.ties[r];
        if (lane == 0 && rank_in < stay) seg_mass += min((u64)ties, stay - rank_in) * w;
        for (uint32_t i0 = s0; i0 < s1; i0 += 32) {
          const uint32_t i = i0 + lane;
          const bool tie = i < s1 && u_of(d_of(key[i])) == ul;
          const uint32_t bal = __ballot_sync(0xffffffffu, tie);
          if (tie && rank_in + __popc(bal & ((1u << lane) - 1u)) >= stay) key[i] = -INFINITY;
          rank_in += __popc(bal);
        }
        break;
      }
      if (level > 1 && uh - ul > span / 2) {
        // the masses' bounds did not separate them (one entry outweighs the others): the exact ones halve the range
        const uint32_t mid = ul + (uh - ul) / 2;
        uint32_t cl = 0;
        u64 ml = 0;
        each([&](uint32_t, float d) {
          if (d < dlow || u_of(d) < ul || u_of(d) > mid) return;
          ++cl;
          ml += mass(d);
        });
        // Every CTA has read what the look before left in ncand and total only once it passes the barrier below, and may
        // still read these sums while a faster one is in the next look, which writes both: hence their own slots.
        push(s.half_count, cta_sum(__reduce_add_sync(0xffffffffu, cl), s.redc, warp, lane));
        push(s.half_mass, cta_sum(warp_sum(ml), s.red, warp, lane));
        cluster.sync();
        uint32_t count = 0;
        u64 sum = 0;
#pragma unroll
        for (int r = 0; r < CL; ++r) {
          count += s.half_count[r];
          sum += s.half_mass[r];
        }
        if (cnt_above + count >= k || above + sum >= thr) {
          uh = umax = mid;
        } else {
          ul = mid + 1;
          cnt_above += count;
          above += sum;
          seg_mass += ml;
        }
      }
      span = uh - ul;
      __syncthreads();
      for (int i = tid; i < kBins; i += kThr) hist[i] = 0;
      __syncthreads();
      done = look(std::false_type{});
    }
    seg_mass = warp_sum(seg_mass);
    if (!struck && cand > 0) {
      // The candidates' key range in kSub parts, with exact counts and masses: the cut falls into one part, and only
      // its members are ranked one against the other.
      for (int i = tid; i < kSub; i += kThr) {
        s.sub_mass[i] = Split{0, 0};
        s.sub_cnt[i] = 0;
      }
      if (tid < kWrp) s.seg_add[tid] = Split{0, 0};
      if (tid == 0) s.cut_n = 0;
      __syncthreads();
      const uint32_t u0 = ul;
      const float per = (float)kSub / ((float)(uh - ul) + 1.0f);
      auto part_of = [&](uint32_t u) { return min(kSub - 1, (int)((float)(u - u0) * per)); };  // ascends with u
      // Every CTA's candidates, a warp or two per CTA.  (mine lies behind `all`, so the copies do not touch what other
      // CTAs read.)
      const bool direct = cand <= 64;  // few enough to be ranked at once
      {
        uint32_t at = 0;
        const int from = warp % CL;
#pragma unroll
        for (int r = 0; r < CL; ++r) at += r < from ? in[r] : 0u;
        const Cand* theirs = cluster.map_shared_rank(mine, from);
        for (uint32_t i = warp / CL * 32 + lane; i < s.ncand[from]; i += 32 * (kWrp / CL)) {
          const Cand x = theirs[i];
          all[at + i] = x;
          if (!direct) {
            const int p = part_of(x.u);
            atomicAdd(&s.sub_cnt[p], 1u);
            s.sub_mass[p].add(x.w);
          }
        }
      }
      __syncthreads();
      // every warp: two parts a lane, cumulative; the first part that reaches top-k or top-p holds the cut
      static_assert(kSub == 64, "two parts a lane");
      const uint32_t c0 = s.sub_cnt[2 * lane], c1 = s.sub_cnt[2 * lane + 1];
      const u64 w0 = s.sub_mass[2 * lane].sum(), w1 = s.sub_mass[2 * lane + 1].sum();
      uint32_t cx = c0 + c1;
      u64 wx = w0 + w1;
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t oc = __shfl_up_sync(0xffffffffu, cx, o);
        const u64 ow = __shfl_up_sync(0xffffffffu, wx, o);
        if (lane >= o) {
          cx += oc;
          wx += ow;
        }
      }
      cx += cnt_above;
      wx += above;
      const bool at1 = cx >= k || wx >= thr, at0 = cx - c1 >= k || wx - w1 >= thr;
      const uint32_t reach = __ballot_sync(0xffffffffu, at1);
      int cut = kSub;  // no part reaches it: all candidates are allowed
      uint32_t cb = cnt_above;
      u64 mb = above;
      if (reach && !direct) {
        const int l = __ffs(reach) - 1;
        const bool low = __shfl_sync(0xffffffffu, at0, l);
        cut = 2 * l + (low ? 0 : 1);
        cb = __shfl_sync(0xffffffffu, low ? cx - c1 - c0 : cx - c1, l);
        mb = __shfl_sync(0xffffffffu, low ? wx - w1 - w0 : wx - w1, l);
      }
      if (!direct) {
        // the cut part's members, in the place of this CTA's candidates (which every CTA has read: the barrier)
        cluster.sync();
        for (uint32_t i = tid; i < cand; i += kThr)
          if (part_of(all[i].u) == cut) {
            const uint32_t at = atomicAdd(&s.cut_n, 1u);
            if (at < kMine) mine[at] = all[i];
          }
        __syncthreads();
      }
      const uint32_t members = direct ? cand : s.cut_n;
      const bool few = members <= kMine;
      const Cand* rivals = few && !direct ? mine : all;
      for (uint32_t i = tid; i < s.ncand[rank]; i += kThr) {
        const Cand me = all[before + i];
        const int p = part_of(me.u);
        bool allowed = p < cut && !direct;
        if (p == cut || direct) {
          uint32_t nb = cb;
          u64 wb = mb;
#pragma unroll 4
          for (uint32_t j = 0; j < (few ? members : cand); ++j) {
            const Cand o = rivals[j];
            const bool ahead = (o.u < me.u || (o.u == me.u && o.idx < me.idx)) && (few || part_of(o.u) == cut);
            nb += ahead;
            wb += ahead ? o.w : 0ull;
          }
          allowed = nb < k && wb < thr;
        }
        if (!allowed)
          key[me.idx - v0] = -INFINITY;
        else
          s.seg_add[(me.idx - v0) / seg].add(me.w);
      }
      __syncthreads();
      seg_mass += s.seg_add[warp].sum();
    }
  }

  // ---- 3. the token
  push(s.kept, cta_sum(seg_mass, s.seg, warp, lane));
  cluster.sync();
  u64 W = 0;
#pragma unroll
  for (int r = 0; r < CL; ++r) W += s.kept[r];
  // floor(u W), exactly: u = m 2^-e with a 53-bit m
  const double u = a.u[row];
  u64 r = 0;
  if (u > 0x1p-64 && u < 1.0) {
    const u64 bits = (u64)__double_as_longlong(u);
    const int e = 1075 - (int)(bits >> 52);  // 53 .. 117
    const u64 m = (bits & 0xfffffffffffffull) | 1ull << 52;
    const u64 ph = __umul64hi(m, W), pl = m * W;
    r = e < 64 ? ph << (64 - e) | pl >> e : ph >> (e - 64);
  } else if (!(u < 1.0)) {
    r = W - 1;  // at or past the end (and NaN): the last allowed token
  }
  u64 base = 0;
  uint32_t owner = 0;
  for (; owner + 1 < (uint32_t)CL && base + s.kept[owner] <= r; ++owner) base += s.kept[owner];
  if (owner != rank) return;
  int ws = 0;
  for (; ws + 1 < kWrp && base + s.seg[ws] <= r; ++ws) base += s.seg[ws];
  // entries of the segment, consecutive ones a thread
  const uint32_t g0 = min(a.slice, ws * seg), g1 = min(a.slice, g0 + seg), per = (seg + kThr - 1) / kThr;
  const uint32_t e0 = min(g1, g0 + tid * per), e1 = min(g1, e0 + per);
  auto mass_at = [&](uint32_t i) -> u64 {
    const float d = d_of(key[i]);
    return d >= dlow && u_of(d) <= umax ? mass(d) : 0ull;
  };
  u64 own = 0;
  for (uint32_t i = e0; i < e1; ++i) own += mass_at(i);
  u64 inc = own;
  for (int o = 1; o < 32; o <<= 1) {
    const u64 x = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += x;
  }
  if (lane == 31) s.red[warp] = inc;
  __syncthreads();
  base += warp_sum(lane < warp ? s.red[lane % kWrp] : 0ull) + inc - own;
  if (own > 0 && base <= r && r < base + own) {
    for (uint32_t i = e0; i < e1; ++i) {
      const u64 w = mass_at(i);
      if (w > 0 && r < base + w) {
        a.token[row] = (int32_t)(v0 + i);
        if (a.prob) a.prob[row] = (float)(exp2((double)d_of(key[i]) * c) / ((double)W * 0x1p-44));
        break;
      }
      base += w;
    }
  }
}

// Few rows: kWide CTAs each, if that many clusters run at once, one CTA on an SM.  (A cluster of more than eight needs
// the kernel's leave, and its SMs in one part of the GPU, so it is asked how many there can be.  1 row of 128,256 with
// top-k and top-p 15.6 -> 14.7 us, with top-p alone 22 -> 18 us; 64 and 256 rows would take 1.7 times as long.)
template <typename S>
bool wide_clusters(uint32_t rows, size_t smem, int sm_count) {
  if ((uint64_t)rows * kWide > (uint64_t)sm_count) return false;
  auto kernel = sample_logits_kernel<S, kWide>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(rows * kWide);
  cfg.blockDim = dim3(kThr);
  cfg.dynamicSmemBytes = smem;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  return n >= (int)rows;
}

template <typename S, int CL>
int launch_sample_logits(SampleArgs a, uint32_t rows, size_t smem, cudaStream_t st) {
  return launch_pdl(sample_logits_kernel<S, CL>, dim3(rows * CL), dim3(kThr), smem, st, a);
}

template <typename S>
int launch_sample_logits(SampleArgs a, uint32_t rows, int sm_count, cudaStream_t st) {
  constexpr int N = 16 / sizeof(S);
  a.vec = (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 && a.ld % N == 0;
  auto memory = [&](int ctas) {
    a.slice = (uint32_t)((ceil_div(a.V, ctas) + N - 1) / N * N);
    a.slice = (a.slice + 3) / 4 * 4;  // four entries a lane, and the tables after the keys stay 16-byte aligned
    return (size_t)a.slice * 4 + 2 * kBins * sizeof(uint32_t);
  };
  size_t smem = memory(kWide);
  CLM_TRY(ensure_smem(sample_logits_kernel<S, kWide>, smem + sizeof(Shared<kWide>)));  // (the limit counts static memory)
  if (wide_clusters<S>(rows, smem, sm_count)) return launch_sample_logits<S, kWide>(a, rows, smem, st);
  smem = memory(kCl);
  CLM_TRY(ensure_smem(sample_logits_kernel<S, kCl>, smem + sizeof(Shared<kCl>)));
  return launch_sample_logits<S, kCl>(a, rows, smem, st);
}

}  // namespace

}  // namespace clm

using namespace clm;

extern "C" int clm_b200_sample_logits(clm_b200_ctx* ctx, const void* d_logits, int dtype, uint32_t rows, uint32_t vocab,
                                      uint64_t ld, const float* d_temperature, const int32_t* d_top_k,
                                      const float* d_top_p, const float* d_min_p, const double* d_uniforms,
                                      int32_t* d_out, float* d_probs, void* stream) {
  CLM_CHECK(ctx != nullptr, CLM_INVALID_ARGUMENT, "null context");
  CLM_CHECK(vocab > 0, CLM_INVALID_ARGUMENT, "empty vocabulary");
  CLM_CHECK(vocab <= kMaxVocab, CLM_OUT_OF_RANGE, "vocabulary too large for sampling");
  CLM_CHECK(ld >= vocab && ld < (1ull << 40), CLM_INVALID_ARGUMENT, "a row stride is smaller than a row");
  CLM_CHECK(dtype >= CLM_DTYPE_F32 && dtype <= CLM_DTYPE_BF16, CLM_INVALID_ARGUMENT, "unknown element type");
  if (rows == 0) return CLM_OK;
  CLM_CHECK(d_logits && d_uniforms && d_out, CLM_INVALID_ARGUMENT, "null buffer");
  CLM_CHECK(rows <= 0x7fffffffu / kCl, CLM_OUT_OF_RANGE, "too many rows");
  SampleArgs a{};
  a.logits = d_logits;
  a.ld = (long long)ld;
  a.V = vocab;
  a.temp = d_temperature;
  a.top_k = d_top_k;
  a.top_p = d_top_p;
  a.min_p = d_min_p;
  a.u = d_uniforms;
  a.token = d_out;
  a.prob = d_probs;
  CLM_SCOPE(ctx);
  cudaStream_t st = pick_stream(ctx, stream);
  if (dtype == CLM_DTYPE_F32) return launch_sample_logits<float>(a, rows, ctx->sm_count, st);
  if (dtype == CLM_DTYPE_F16) return launch_sample_logits<__half>(a, rows, ctx->sm_count, st);
  return launch_sample_logits<__nv_bfloat16>(a, rows, ctx->sm_count, st);
}
