// Next-token sampling from given uniform numbers: temperature, top-k, top-p and min-p per row, one launch.
//
//   w_i = exp((x_i - max) / T);  in descending order of x (equal ones: lowest index first)
//     top-k keeps what is not below the k-th value, top-p the longest prefix with sum(w) <= p sum(all w) (at least one token),
//     min-p what has w_i >= m;  the token is the first index, in the vocabulary's order, with sum_{kept, j <= i} w_j > u sum_kept w.
//
// A row belongs to a cluster of up to sixteen CTAs, each with a contiguous slice of the logits in shared memory: they are read from
// global memory once.  Weights are 44-bit fixed-point numbers formed in double precision (2^-44 of the largest), so sums are
// integers: exact in any order, equal from run to run, and a prefix ends where its definition says.  All filters are one cut (key, index)
// in the descending order.  It is found by a histogram over 1/32 octave of weight (counts for k, sums for p), whose
// bins every CTA adds up through distributed shared memory; the candidates of the one bin that the cut falls into are collected by every CTA
// and divided further by the bits of their keys until few are left, which are ranked against each other.  Should they be too many to be
// collected (equal logits), the whole slices are divided again, down to a single value whose ties are counted in index order.
//
// A row is bound by the latency of its stages: 17.5 us for 65536 fp32 logits with top-p 0.95 on 16 CTAs (read 1.4, maximum 1.4, histogram 2.6, its
// exchange and border 4.4, candidates 2, ranking 2.5, kept list 1.5, token 1.7), where the bytes would take 0.04.  A batch of 64 such rows with settings of
// their own (4 CTAs each, two per SM) takes 41.3 us: 14 of them are the histogram pass, bound by the instructions that form the weights (atomics 3,
// the table 1, both measured by leaving them out).  Differences of two logits and their exponents are formed in double precision: either may lie outside
// fp32, and the products' common rounding, 2^-53 of max / T, stays below a weight's last bit for logits of up to some hundreds of temperatures.
#include <cooperative_groups.h>

#include <utility>

#include "common.cuh"

namespace b200 {
namespace cg = cooperative_groups;

constexpr int SP_THREADS = 512, SP_WARPS = SP_THREADS / 32, SP_BINS = 512, SP_CAND = 1024, SP_FEW = 128, SP_MAX_CTAS = 16, SP_TAB = 256, SP_LIST = 512;
constexpr int SP_SEG = SP_THREADS / SP_FEW;         // threads that rank a candidate
constexpr float SP_BINS_PER_OCTAVE = 32.f;
constexpr int SP_MAX_SMEM = 180 * 1024;             // for the slice
constexpr int SP_ONE = 44;                          // a weight of 1 is 2^44; 2^20 of them fit the sums (a row has 327680 at most)
static_assert(SP_BINS == SP_THREADS, "a bin per thread");

struct SampleParams {
  const void* logits;                               // [B, V], row pitch ld
  long long ld;
  int V, per;                                       // per: slice of a CTA, a multiple of SP_THREADS
  const float* uniform;
  const float *temperature, *top_p, *min_p;         // [B]; null: the value below
  const int* top_k;
  float t, p, m;
  int k;
  long long* out;
};

struct SampleHist {
  uint32_t cnt[SP_BINS];
  struct alignas(8) { uint32_t lo, hi; } mass[SP_BINS];     // sums of weights as two words
};
struct SampleShared {
  SampleHist hist;                                  // this slice
  uint32_t key[SP_CAND], idx[SP_CAND];              // candidates of this slice
  union {
    struct {
      uint32_t key[SP_CAND], idx[SP_CAND];          // of the row, SP_CAND / CTAs places for each slice; key 0: none
      union {
        SampleHist sub;
        struct {                                    // the last few: keys, indices, weights, and what each quarter of them puts in front
          uint32_t key[SP_FEW], idx[SP_FEW];
          unsigned long long w[SP_FEW], sum[SP_SEG][SP_FEW];
          uint32_t rank[SP_SEG][SP_FEW];
        } few;
      } u;
    } all;
    uint16_t list[SP_WARPS][SP_LIST];               // kept elements of a warp's part, in order
  } w;
  double tab[SP_TAB];                               // 2^(44 - i / 256)
  unsigned long long red[SP_WARPS], red2[SP_WARPS];
  unsigned long long xch[2][SP_MAX_CTAS];           // what the CTAs of the cluster tell each other
  uint32_t xa[2][SP_MAX_CTAS], xb[2][SP_MAX_CTAS];
  uint32_t ncand, nsel;
  int found, found2, cut_idx;
  uint32_t cut_k, cut_p;
  unsigned long long before[2];
};

__device__ __forceinline__ uint32_t sp_key(float x) {
  const uint32_t b = __float_as_uint(x);
  return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float sp_unkey(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu)); }

__device__ __forceinline__ unsigned long long warp_sum64(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ unsigned long long warp_scan64(unsigned long long v) {   // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long u = __shfl_up_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) >= o) v += u;
  }
  return v;
}

// w to a bin of a histogram; the carry of the lower word goes to the upper one, so the sum is exact whatever the order.
__device__ __forceinline__ void sp_add(SampleHist& h, int bin, unsigned long long w) {
  const uint32_t l = static_cast<uint32_t>(w), old = atomicAdd(&h.mass[bin].lo, l);
  const uint32_t up = static_cast<uint32_t>(w >> 32) + (old + l < old ? 1u : 0u);
  if (up) atomicAdd(&h.mass[bin].hi, up);
}
__device__ __forceinline__ unsigned long long sp_mass(const SampleHist& h, int bin) { return *reinterpret_cast<const unsigned long long*>(&h.mass[bin]); }

struct SampleScale {
  float mx;
  double c, mxc;                                    // log2(e) / T; max times that
};
// 2^-y, y = (max - v) log2(e) / T = a + i / 256 + r, in units of 2^-44.
__device__ __forceinline__ unsigned long long sp_weight_inline(float v, float mx, double c, double mxc, const double* tab) {
  const double y = fma(-static_cast<double>(v), c, mxc);
  const double big = 6755399441055744.0 / SP_TAB;   // 1.5 * 2^52 / 256: adding it leaves round(256 y) in the low bits
  const double z = y + big;
  const int q = __double2loint(z);
  const double r = y - (z - big);                   // |r| <= 2^-9; 2^-r = 1 - z + z^2 / 2 - z^3 / 6, z = r ln 2, to 2e-13
  const double e = fma(r, fma(r, fma(r, -0.055504108664821580, 0.24022650695910071), -0.69314718055994531), 1.0);
  const double f = fma(tab[q & (SP_TAB - 1)], e, 4503599627370496.0);           // 2^52: the low bits are the rounded integer
  const unsigned long long w = (static_cast<unsigned long long>(__double_as_longlong(f)) & 0xFFFFFFFFFFFFFull) >> (q >> 8 & 63);
  return v == mx ? 1ull << SP_ONE : y < SP_ONE + 1. ? w : 0ull;     // (infinities, too; y because mx - v and c may leave fp32)
}
// Not inlined where speed does not ask for it: a row runs through every stage of the kernel once, and with eight copies of this in it the
// fetching of instructions took a third of its time.
__device__ __noinline__ unsigned long long sp_weight(float v, float mx, double c, double mxc, const double* tab) {
  return sp_weight_inline(v, mx, c, mxc, tab);
}
static_assert(SP_TAB == 256, "shifts by eight above");

template <typename T>
__global__ void __launch_bounds__(SP_THREADS, 2)
sample_kernel(const SampleParams p) {
  extern __shared__ float sx[];                     // logits of the slice, NaN as -inf; element i at i + i / 32
  __shared__ SampleShared s;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int row = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int lo = rank * p.per, n = max(0, min(p.per, p.V - lo));
  const int chunk = p.per / SP_WARPS, each = chunk / 32;        // warps own contiguous parts of the slice, lanes parts of those
  const int w0 = min(n, warp * chunk), w1 = min(n, w0 + chunk);
  int phase = 0;                                    // exchanges alternate between two places
  auto at = [&](int i) -> float& { return sx[i + (i >> 5)]; };  // both orders of access meet no bank twice

  auto started = cluster.barrier_arrive();          // before the first access to another CTA's memory it has to be running
  if (tid < SP_TAB) s.tab[tid] = exp2(static_cast<double>(SP_ONE) - tid / static_cast<double>(SP_TAB));
  auto clear = [&]() {                              // before a histogram, and before candidates arrive
    s.hist.cnt[tid] = s.hist.mass[tid].lo = s.hist.mass[tid].hi = 0;
    for (int i = tid; i < SP_CAND; i += SP_THREADS) s.w.all.key[i] = 0;
  };
  clear();
  pdl_trigger();
  pdl_wait();
  const T* x = static_cast<const T*>(p.logits) + static_cast<long long>(row) * p.ld + lo;
  const float T_ = p.temperature ? p.temperature[row] : p.t;
  const float top_p = p.top_p ? p.top_p[row] : p.p, min_p = fminf(p.min_p ? p.min_p[row] : p.m, 1.f);
  const int top_k = p.top_k ? p.top_k[row] : p.k;
  const float u = p.uniform[row];

  // ---- the slice, its maximum and where it is first
  uint32_t best = 0, where = 0;
  auto take = [&](int i, float v) {
    v = v == v ? v + 0.f : -INFINITY;               // -0 and 0 are one value
    at(i) = v;
    const uint32_t k = sp_key(v);
    if (k > best) { best = k; where = lo + i; }     // a thread meets its elements in index order
  };
  if (sizeof(T) == 2 && !(reinterpret_cast<uintptr_t>(x) & 3)) {
#pragma unroll 4
    for (int i = tid; i < n / 2; i += SP_THREADS) {
      const float2 f = unpack_bf16x2(__ldg(reinterpret_cast<const uint32_t*>(x) + i));
      take(2 * i, f.x);
      take(2 * i + 1, f.y);
    }
    if ((n & 1) && tid == 0) take(n - 1, static_cast<float>(x[n - 1]));
  } else {
#pragma unroll 8
    for (int i = tid; i < n; i += SP_THREADS) take(i, static_cast<float>(x[i]));
  }
  // larger key first, then the lower index
  unsigned long long top = (static_cast<unsigned long long>(best) << 32) | (0xFFFFFFFFu - where);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) s.red[warp] = top;
  __syncthreads();
  cluster.barrier_wait(std::move(started));
  if (warp == 0) {
    top = lane < SP_WARPS ? s.red[lane] : 0ull;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    top = __shfl_sync(0xffffffffu, top, 0);
    if (lane < C) cluster.map_shared_rank(&s, lane)->xch[phase][rank] = top;
  }
  cluster.sync();
  top = 0;
  for (int c = 0; c < C; ++c) top = max(top, s.xch[phase][c]);
  phase ^= 1;
  const float mx = sp_unkey(static_cast<uint32_t>(top >> 32));
  const bool none = mx == -INFINITY;
  if (none || !(T_ > 0.f)) {                        // nothing to choose from / greedy
    if (rank == 0 && tid == 0) p.out[row] = none ? -1ll : static_cast<long long>(0xFFFFFFFFu - static_cast<uint32_t>(top));
    return;                                         // no CTA touches another's memory after the barrier
  }

  SampleScale sc;
  sc.mx = mx;
  sc.c = 1.4426950408889634 / static_cast<double>(T_);
  sc.mxc = static_cast<double>(mx) * sc.c;
  const float cf = static_cast<float>(sc.c);        // for bins, which do not have to be exact
  auto weight = [&](float v) { return sp_weight(v, sc.mx, sc.c, sc.mxc, s.tab); };

  // ---- the cut: kept are keys above cut_key, and those equal to it with an index up to cut_idx
  uint32_t cut_key = 0;
  int cut_idx = INT_MAX;
  auto cut = [&](uint32_t key, int idx) {
    if (key > cut_key || (key == cut_key && idx < cut_idx)) { cut_key = key; cut_idx = idx; }
  };
  if (min_p > 0.f) {
    // an infinite temperature drops nothing that weighs something (and inf - inf would be no threshold)
    const double thr = isinf(T_) ? -INFINITY : static_cast<double>(mx) + static_cast<double>(T_) * log(static_cast<double>(min_p));
    float f = static_cast<float>(thr);
    uint32_t k = sp_key(f + 0.f);
    if (static_cast<double>(f) < thr) ++k;          // the least float that is not below
    cut(k, INT_MAX);
  }
  bool by_k = top_k > 0 && top_k < p.V, by_p = top_p > 0.f && top_p < 1.f;
  unsigned long long limit = 0, mass_before = 0, cnt_before = 0;    // largest prefix sum; what lies in front of the present subset

  // The first bin in which a limit is passed (SP_BINS: none), from the counts and sums of thread's bin; moves the sums in front along.
  auto crossing = [&](uint32_t cnt_b, unsigned long long mass_b, bool first) -> int {
    unsigned long long cs = by_k ? warp_scan64(cnt_b) : 0ull, ms = by_p ? warp_scan64(mass_b) : 0ull;
    if (lane == 31) { s.red[warp] = cs; s.red2[warp] = ms; }
    if (tid == 0) { s.found = SP_BINS; s.found2 = SP_BINS; s.nsel = 0; }
    __syncthreads();
    unsigned long long total = 0;
    for (int w = 0; w < SP_WARPS; ++w) {
      if (w < warp) { cs += s.red[w]; ms += s.red2[w]; }
      total += s.red2[w];
    }
    cs += cnt_before;
    ms += mass_before;
    if (first) limit = static_cast<unsigned long long>(static_cast<double>(top_p) * static_cast<double>(total));
    const bool past_k = by_k && cs >= static_cast<unsigned long long>(top_k), past_p = by_p && ms > limit;
    const uint32_t vk = __ballot_sync(0xffffffffu, past_k), vp = __ballot_sync(0xffffffffu, past_p);
    if (lane == 0 && vk) atomicMin(&s.found, 32 * warp + __ffs(vk) - 1);
    if (lane == 0 && vp) atomicMin(&s.found2, 32 * warp + __ffs(vp) - 1);
    __syncthreads();
    const int bk = s.found, bp = s.found2, hit = min(bk, bp);
    if (hit == SP_BINS) return hit;
    by_k = by_k && bk == hit;
    by_p = by_p && bp == hit;
    if (tid == hit) { s.before[0] = cs - cnt_b; s.before[1] = ms - mass_b; }
    __syncthreads();
    cnt_before = s.before[0];
    mass_before = s.before[1];
    return hit;
  };

  if (by_k || by_p) {
    const float bin_scale = cf * SP_BINS_PER_OCTAVE;
    bool first = true;
    uint32_t kmin = 0, kmax = 0xFFFFFFFFu;
    int shift = 0;
    auto bin_of = [&](float v) -> int {             // does not rise with v
      if (first) return min(SP_BINS - 1, static_cast<int>((mx - v) * bin_scale));
      const uint32_t k = sp_key(v);
      return k < kmin || k > kmax ? -1 : static_cast<int>((kmax - k) >> shift);
    };
    while (true) {
      // most tokens of a vocabulary are improbable and share the last bin: they are added up in registers
      uint32_t rest = 0;
      unsigned long long rest_w = 0;
#pragma unroll 4
      for (int i = w0 + lane; i < w1; i += 32) {
        const float v = at(i);
        const int bin = bin_of(v);
        const unsigned long long w = by_p ? sp_weight_inline(v, sc.mx, sc.c, sc.mxc, s.tab) : 0ull;
        if (bin == SP_BINS - 1) {
          ++rest;
          rest_w += w;
        } else if (bin >= 0) {
          if (by_k) atomicAdd(&s.hist.cnt[bin], 1u);
          if (w) sp_add(s.hist, bin, w);
        }
      }
      rest = __reduce_add_sync(0xffffffffu, rest);
      rest_w = warp_sum64(rest_w);
      if (lane == 0 && rest) {
        atomicAdd(&s.hist.cnt[SP_BINS - 1], rest);
        sp_add(s.hist, SP_BINS - 1, rest_w);
      }
      if (tid == 0) s.ncand = 0;
      cluster.sync();
      {                                             // the slices' sums of a share of the bins, handed to every CTA: 8 KB to move, not 64
        const int q = tid & (C - 1), bin = rank * (SP_BINS / C) + tid / C;
        const SampleHist& h = cluster.map_shared_rank(&s, q)->hist;
        uint32_t cnt = h.cnt[bin];
        unsigned long long mass = sp_mass(h, bin);
        for (int o = C >> 1; o > 0; o >>= 1) {
          cnt += __shfl_xor_sync(0xffffffffu, cnt, o);
          mass += __shfl_xor_sync(0xffffffffu, mass, o);
        }
        SampleHist& sum = cluster.map_shared_rank(&s, q)->w.all.u.sub;
        sum.cnt[bin] = cnt;
        *reinterpret_cast<unsigned long long*>(&sum.mass[bin]) = mass;
      }
      cluster.sync();
      const uint32_t cnt_b = s.w.all.u.sub.cnt[tid];
      const unsigned long long mass_b = sp_mass(s.w.all.u.sub, tid);
      const int hit = crossing(cnt_b, mass_b, first);
      if (hit == SP_BINS) break;                    // the rest passes no limit (the same in all CTAs)
      // ---- the bin's candidates: listed, then handed to every CTA
#pragma unroll 2
      for (int i = w0 + lane; i < w1; i += 32) {
        const float v = at(i);
        if (bin_of(v) == hit) {
          const uint32_t slot = atomicAdd(&s.ncand, 1u);
          if (slot < SP_CAND) { s.key[slot] = sp_key(v); s.idx[slot] = lo + i; }
        }
      }
      __syncthreads();
      const uint32_t room = SP_CAND / C, found = s.ncand;
      for (uint32_t i = tid; i < C * min(found, room); i += SP_THREADS) {
        SampleShared* r = cluster.map_shared_rank(&s, i & (C - 1));
        const uint32_t j = i / C;
        r->w.all.key[rank * room + j] = s.key[j];
        r->w.all.idx[rank * room + j] = s.idx[j];
      }
      if (tid < C) cluster.map_shared_rank(&s, tid)->xa[phase][rank] = found;
      cluster.sync();
      uint32_t left = 0, most = 0;
      for (int q = 0; q < C; ++q) {
        left += s.xa[phase][q];
        most = max(most, s.xa[phase][q]);
      }
      phase ^= 1;
      if (most <= room) {
        // ---- divided by the bits of their keys until few are left
        kmin = 1;
        kmax = 0xFFFFFFFFu;
        while (left > SP_FEW) {
          uint32_t a = 0xFFFFFFFFu, z = 0;
          for (int i = tid; i < SP_CAND; i += SP_THREADS) {
            const uint32_t k = s.w.all.key[i];
            if (k >= kmin && k <= kmax) { a = min(a, k); z = max(z, k); }
          }
          a = __reduce_min_sync(0xffffffffu, a);
          z = __reduce_max_sync(0xffffffffu, z);
          if (lane == 0) { s.red[warp] = a; s.red2[warp] = z; }
          s.w.all.u.sub.cnt[tid] = s.w.all.u.sub.mass[tid].lo = s.w.all.u.sub.mass[tid].hi = 0;
          __syncthreads();
          for (int w = 0; w < SP_WARPS; ++w) { a = min(a, static_cast<uint32_t>(s.red[w])); z = max(z, static_cast<uint32_t>(s.red2[w])); }
          kmin = a;
          kmax = z;
          if (kmin == kmax) break;                  // equal logits
          shift = max(0, 32 - __clz(kmax - kmin) - 9);
          for (int i = tid; i < SP_CAND; i += SP_THREADS) {
            const uint32_t k = s.w.all.key[i];
            if (k < kmin || k > kmax) continue;
            const int bin = static_cast<int>((kmax - k) >> shift);
            atomicAdd(&s.w.all.u.sub.cnt[bin], 1u);
            if (by_p) sp_add(s.w.all.u.sub, bin, weight(sp_unkey(k)));
          }
          __syncthreads();
          const int sub = crossing(s.w.all.u.sub.cnt[tid], sp_mass(s.w.all.u.sub, tid), false);
          left = s.w.all.u.sub.cnt[sub];            // there is one: the bin passes the limit
          const uint32_t high = kmax - (static_cast<uint32_t>(sub) << shift);
          kmin = max(kmin, high - ((1u << shift) - 1));
          kmax = high;
          __syncthreads();                          // sub has been read
        }
        if (tid == 0) { s.nsel = 0; s.found = 0; s.cut_k = 0; s.cut_idx = INT_MAX; }
        __syncthreads();
        if (left <= SP_FEW) {
          // ---- ranked against each other: SP_SEG threads per candidate find its rank and the weights in front of it
          auto& few = s.w.all.u.few;
          for (int i = tid; i < SP_CAND; i += SP_THREADS) {
            const uint32_t k = s.w.all.key[i];
            if (k >= kmin && k <= kmax) {
              const uint32_t slot = atomicAdd(&s.nsel, 1u);
              few.key[slot] = k;
              few.idx[slot] = s.w.all.idx[i];
              few.w[slot] = by_p ? weight(sp_unkey(k)) : 0ull;
            }
          }
          __syncthreads();
          const uint32_t i = tid % SP_FEW, seg = tid / SP_FEW;
          uint32_t k = 0, d = 0;
          if (i < left) {
            k = few.key[i];
            d = few.idx[i];
            uint32_t r = 0;
            unsigned long long sum = 0;
#pragma unroll 2
            for (uint32_t j = seg; j < left; j += SP_SEG) {
              const bool front = few.key[j] > k || (few.key[j] == k && few.idx[j] < d);
              r += front;
              sum += front ? few.w[j] : 0ull;
            }
            few.rank[seg][i] = r;
            few.sum[seg][i] = sum;
          }
          __syncthreads();
          uint32_t r = 0;
          unsigned long long run = mass_before;
          if (tid < left) {
            for (int q = 0; q < SP_SEG; ++q) { r += few.rank[q][tid]; run += few.sum[q][tid]; }
            if (by_k && r == top_k - cnt_before - 1) s.cut_k = k;                 // ties with the k-th stay
            if (by_p && run + few.w[tid] <= limit) atomicMax(&s.found, static_cast<int>(r) + 1);
          }
          __syncthreads();
          if (by_k) cut(s.cut_k, INT_MAX);
          if (by_p) {
            const int keep = s.found ? s.found : mass_before == 0 ? 1 : 0;        // the most probable token stays
            if (tid < left && r == static_cast<uint32_t>(max(keep, 1) - 1)) { s.cut_p = k; s.cut_idx = static_cast<int>(d) - (keep ? 0 : 1); }
            __syncthreads();
            cut(s.cut_p, s.cut_idx);
          }
        } else {
          // ---- many equal ones: they stay in index order
          const unsigned long long w = by_p ? weight(sp_unkey(kmin)) : 0ull;
          unsigned long long keep = left;
          if (w) keep = limit > mass_before ? min(keep, (limit - mass_before) / w) : 0ull;
          if (keep == 0 && mass_before == 0) keep = 1;
          if (keep < left) {
            if (keep == 0 && tid == 0) s.cut_idx = -1;
            for (int i = tid; i < SP_CAND; i += SP_THREADS) {
              if (s.w.all.key[i] != kmin) continue;
              uint32_t r = 0;
              for (int j = 0; j < SP_CAND; ++j) r += s.w.all.key[j] == kmin && s.w.all.idx[j] < s.w.all.idx[i];
              if (r + 1 == keep) s.cut_idx = static_cast<int>(s.w.all.idx[i]);
            }
          }
          __syncthreads();
          cut(kmin, s.cut_idx);
        }
        break;
      }
      // ---- too many: divide the bin by the bits of its keys
      uint32_t a = 0xFFFFFFFFu, z = 0;
      for (int i = w0 + lane; i < w1; i += 32)
        if (bin_of(at(i)) == hit) {
          a = min(a, sp_key(at(i)));
          z = max(z, sp_key(at(i)));
        }
      a = __reduce_min_sync(0xffffffffu, a);
      z = __reduce_max_sync(0xffffffffu, z);
      if (lane == 0) { s.red[warp] = a; s.red2[warp] = z; }
      __syncthreads();
      if (tid < C) {
        unsigned long long a2 = 0xFFFFFFFFull, z2 = 0;
        for (int w = 0; w < SP_WARPS; ++w) { a2 = min(a2, s.red[w]); z2 = max(z2, s.red2[w]); }
        SampleShared* r = cluster.map_shared_rank(&s, tid);
        r->xa[phase][rank] = static_cast<uint32_t>(a2);
        r->xb[phase][rank] = static_cast<uint32_t>(z2);
      }
      clear();                                      // all have read and are done with the present lists
      cluster.sync();
      kmin = 0xFFFFFFFFu;
      kmax = 0;
      for (int q = 0; q < C; ++q) { kmin = min(kmin, s.xa[phase][q]); kmax = max(kmax, s.xb[phase][q]); }
      phase ^= 1;
      first = false;
      if (kmin < kmax) {
        shift = max(0, 32 - __clz(kmax - kmin) - 9);            // 2^9 bins
        continue;
      }
      // ---- one value: its ties stay in index order
      const unsigned long long w = weight(sp_unkey(kmin));
      const unsigned long long cand = left;
      unsigned long long keep = cand;
      if (by_p && w) keep = limit > mass_before ? min(keep, (limit - mass_before) / w) : 0ull;
      if (keep == 0 && mass_before == 0) keep = 1;
      cut(kmin, keep == 0 ? -1 : INT_MAX);
      if (keep && keep < cand) {                    // the index of the last one that stays
        uint32_t mine = 0;
        for (int i = w0 + lane; i < w1; i += 32) mine += sp_key(at(i)) == kmin;
        mine = __reduce_add_sync(0xffffffffu, mine);
        if (lane == 0) s.red[warp] = mine;
        __syncthreads();
        if (tid < C) {
          unsigned long long m = 0;
          for (int q = 0; q < SP_WARPS; ++q) m += s.red[q];
          cluster.map_shared_rank(&s, tid)->xa[phase][rank] = static_cast<uint32_t>(m);
        }
        cluster.sync();
        unsigned long long togo = keep;             // ties up to and with the last one, from this warp's first on
        bool here = true;
        for (int q = 0; q < rank; ++q) { here = here && togo > s.xa[phase][q]; togo -= s.xa[phase][q]; }
        for (int q = 0; q < warp; ++q) { here = here && togo > s.red[q]; togo -= s.red[q]; }
        if (here && togo <= mine) {
          for (int i0 = w0; i0 < w1; i0 += 32) {
            const bool eq = i0 + lane < w1 && sp_key(at(i0 + lane)) == kmin;
            const uint32_t vote = __ballot_sync(0xffffffffu, eq);
            const uint32_t m = __popc(vote);
            if (togo <= m) {
              if (eq && __popc(vote & ((2u << lane) - 1)) == static_cast<int>(togo))
                for (int q = 0; q < C; ++q) cluster.map_shared_rank(&s, q)->xb[phase][0] = lo + i0 + lane;
              break;
            }
            togo -= m;
          }
        }
        cluster.sync();
        cut(kmin, static_cast<int>(s.xb[phase][0]));
        phase ^= 1;
      }
      break;
    }
  }

  // ---- sums of the kept weights in index order.  Where a cut leaves few, a warp lists them first; else lanes own neighbouring elements.
  auto keep = [&](int i) {
    const uint32_t k = sp_key(at(i));
    return k > cut_key || (k == cut_key && lo + i <= cut_idx);
  };
  __syncthreads();                                  // the candidates make room for the lists
  uint16_t* list = s.w.list[warp];
  int listed = -1;                                  // kept elements; -1: not listed
  if (cut_key) {
    listed = 0;
#pragma unroll 2
    for (int i0 = w0; i0 < w1; i0 += 32) {
      const bool k = i0 + lane < w1 && keep(i0 + lane);
      const uint32_t vote = __ballot_sync(0xffffffffu, k);
      const int to = listed + __popc(vote & ((1u << lane) - 1));
      if (k && to < SP_LIST) list[to] = static_cast<uint16_t>(i0 + lane);
      listed += __popc(vote);
    }
    if (listed > SP_LIST) listed = -1;
    __syncwarp();
  }
  const int l0 = min(w1, w0 + lane * each), l1 = min(w1, l0 + each);
  unsigned long long mine = 0;
  if (listed >= 0) {
    for (int i = lane; i < listed; i += 32) mine += weight(at(list[i]));
  } else {
#pragma unroll 1
    for (int i = l0; i < l1; ++i) {
      if (keep(i)) mine += weight(at(i));
    }
  }
  const unsigned long long upto = warp_scan64(mine);            // with this lane
  if (lane == 31) s.red[warp] = upto;
  __syncthreads();
  if (tid < C) {
    unsigned long long m = 0;
    for (int q = 0; q < SP_WARPS; ++q) m += s.red[q];
    cluster.map_shared_rank(&s, tid)->xch[phase][rank] = m;
  }
  cluster.sync();
  unsigned long long sum = 0, front = 0;
  for (int q = 0; q < C; ++q) {
    if (q < rank) front += s.xch[phase][q];
    sum += s.xch[phase][q];
  }
  for (int q = 0; q < warp; ++q) front += s.red[q];
  const unsigned long long target = min(static_cast<unsigned long long>(fmax(0.0, static_cast<double>(u) * static_cast<double>(sum))), sum - 1);
  const uint32_t vote = __ballot_sync(0xffffffffu, front + upto > target);
  if (front > target || !vote) return;
  // one warp of the row: 32 elements of its list, or of the lane that the number falls into, at a time
  int from = 0, to = listed;
  if (listed < 0) {
    const int owner = __ffs(vote) - 1;
    front += __shfl_sync(0xffffffffu, upto - mine, owner);
    from = __shfl_sync(0xffffffffu, l0, owner);
    to = __shfl_sync(0xffffffffu, l1, owner);
  }
  for (int i0 = from; i0 < to; i0 += 32) {
    const int i = min(i0 + lane, to - 1), e = listed >= 0 ? list[i] : i;
    const unsigned long long w = weight(at(e));
    const unsigned long long run = front + warp_scan64(i0 + lane < to && (listed >= 0 || keep(e)) ? w : 0ull);
    const uint32_t v = __ballot_sync(0xffffffffu, run > target);
    if (v) {
      if (lane == __ffs(v) - 1) p.out[row] = lo + e;
      return;
    }
    front = __shfl_sync(0xffffffffu, run, 31);
  }
}

}  // namespace b200

using namespace b200;

// CTAs per row: as many as the machine holds at a time (two per SM) and slices of more than 1024 elements allow; at most 40960 to a slice.  For few rows
// a cluster beyond the portable size, on a device that schedules one (`wide`).
B200_API int b200_sample_ctas(int B, int V, int sms, int wide) {
  int C = 1;
  while (C < 8 && ((V + C - 1) / C > 40960 || (static_cast<long long>(B) * C <= sms && (V + C - 1) / C > 1024))) C *= 2;
  if (C == 8 && wide && B <= 4 && (V + C - 1) / C > 2048) C = 16;
  return C;
}
static int sample_per(int V, int C) { return ((V + C - 1) / C + SP_THREADS - 1) / SP_THREADS * SP_THREADS; }
static int sample_smem(int per) { return (per + per / 32) * 4; }

// logits: [B, V] (pitch ld elements), bf16 or fp32; uniform: [B]; per-row tensors may be null (then t, k, p, m hold); out: int64 [B].
B200_API int b200_sample(const SampleParams* a, int B, int is_bf16, void* stream) {
  SampleParams p = *a;
  if (B <= 0 || p.V <= 0 || p.V > 8 * 40960 || p.ld < p.V || !p.logits || !p.uniform || !p.out) return -1;
  auto kern = is_bf16 ? sample_kernel<__nv_bfloat16> : sample_kernel<float>;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -3;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = 16;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.blockDim = dim3(SP_THREADS);
  cfg.attrs = at;
  struct Device { int sms, wide; };
  static Device known[64][2] = {};                  // the same for every call: threads may find them twice
  Device& d = known[dev][is_bf16 != 0];
  if (!d.sms) {
    Device x = {};
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SP_MAX_SMEM) != cudaSuccess ||
        cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
        cudaDeviceGetAttribute(&x.sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      return -4;
    cfg.gridDim = dim3(16);
    cfg.dynamicSmemBytes = sample_smem(sample_per(8 * 40960, 16));              // of the longest rows
    cfg.numAttrs = 1;
    int clusters = 0;
    if (cudaOccupancyMaxActiveClusters(&clusters, kern, &cfg) != cudaSuccess) cudaGetLastError();       // none, then
    x.wide = clusters > 0;
    d.wide = x.wide;
    d.sms = x.sms;
  }
  const int C = b200_sample_ctas(B, p.V, d.sms, d.wide);
  p.per = sample_per(p.V, C);
  const int smem = sample_smem(p.per);
  if (smem > SP_MAX_SMEM || static_cast<long long>(B) * C > (1ll << 31) - 1) return -2;
  cfg.gridDim = dim3(static_cast<unsigned>(B * C));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  at[0].val.clusterDim.x = C;
  cfg.numAttrs = g_b200_pdl ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, p) == cudaSuccess ? 0 : -10;
}
