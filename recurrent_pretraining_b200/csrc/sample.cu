// Next-token sampling from given uniform numbers: temperature, top-k, top-p and min-p per row, one launch.
//
//   w_i = exp((x_i - max) / T);  in descending order of x (equal ones: lowest index first)
//     top-k keeps what is not below the k-th value, top-p the longest prefix with sum(w) <= p sum(all w) (at least one token),
//     min-p what has w_i >= m;  the token is the first index, in the vocabulary's order, with sum_{kept, j <= i} w_j > u sum_kept w.
//
// A row belongs to a cluster of up to eight CTAs, each with a contiguous slice of the logits in shared memory: they are read from
// global memory once.  Weights are 44-bit fixed-point numbers formed in double precision (2^-44 of the largest), so sums are
// integers: exact in any order, equal from run to run, and a prefix ends where its definition says.  All filters are one cut (key, index)
// in the descending order.  It is found by a histogram over 1/16 octave of weight (counts for k, sums for p), whose
// bins the CTAs add up through distributed shared memory; the candidates of the one bin that the cut falls into are ranked against each
// other.  Should they be too many (equal logits), the bin is divided again by the bits of its keys, down to a single value whose ties
// are counted in index order.
#include <cooperative_groups.h>

#include <utility>

#include "common.cuh"

namespace b200 {
namespace cg = cooperative_groups;

constexpr int SP_THREADS = 512, SP_WARPS = SP_THREADS / 32, SP_BINS = 512, SP_CAND = 1024, SP_MAX_CTAS = 8, SP_TAB = 256;
constexpr float SP_BINS_PER_OCTAVE = 16.f;
constexpr int SP_ONE = 44;                          // a weight of 1 is 2^44; 2^18 of them fit the sums

struct SampleParams {
  const void* logits;                               // [B, V], row pitch ld
  long long ld;
  int V, per;                                       // per: slice of a CTA, a multiple of 8
  const float* uniform;
  const float *temperature, *top_p, *min_p;         // [B]; null: the value below
  const int* top_k;
  float t, p, m;
  int k;
  long long* out;
};

struct SampleShared {
  union {
    struct { uint32_t cnt[SP_BINS], lo[SP_BINS], hi[SP_BINS]; } h;             // this slice
    struct { uint32_t key[SP_CAND], idx[SP_CAND]; } c;
  } a;
  union {
    struct { uint32_t cnt[SP_BINS]; unsigned long long mass[SP_BINS]; } h;     // the whole row
    unsigned long long sorted[SP_CAND];
  } b;
  double tab[SP_TAB];                               // 2^(44 - i / 256)
  unsigned long long red[SP_WARPS], red2[SP_WARPS];
  unsigned long long xch[2][SP_MAX_CTAS];           // what the CTAs of the cluster tell each other
  uint32_t xa[2][SP_MAX_CTAS], xb[2][SP_MAX_CTAS];
  uint32_t ncand;
  int found, found2;
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

template <typename T>
__global__ void __launch_bounds__(SP_THREADS)
sample_kernel(const SampleParams p) {
  extern __shared__ float sx[];                     // [per] logits of the slice, NaN as -inf
  __shared__ SampleShared s;
  cg::cluster_group cluster = cg::this_cluster();
  const int C = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int row = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int lo = rank * p.per, n = max(0, min(p.per, p.V - lo));
  const int chunk = p.per / SP_WARPS;               // warps own contiguous parts of the slice
  const int w0 = min(n, warp * chunk), w1 = min(n, w0 + chunk);
  int phase = 0;                                    // exchanges alternate between two places

  auto started = cluster.barrier_arrive();          // before the first access to another CTA's memory it has to be running
  if (tid < SP_TAB) s.tab[tid] = exp2(static_cast<double>(SP_ONE) - tid / static_cast<double>(SP_TAB));
  pdl_trigger();
  pdl_wait();
  const T* x = static_cast<const T*>(p.logits) + static_cast<long long>(row) * p.ld + lo;
  const float T_ = p.temperature ? p.temperature[row] : p.t;
  const float top_p = p.top_p ? p.top_p[row] : p.p, min_p = fminf(p.min_p ? p.min_p[row] : p.m, 1.f);
  const int top_k = p.top_k ? p.top_k[row] : p.k;
  const float u = p.uniform[row];

  // ---- the slice, its maximum and where it is first
  uint32_t best = 0, at = 0;
  auto take = [&](int i, float v) {
    v = v == v ? v + 0.f : -INFINITY;               // -0 and 0 are one value
    sx[i] = v;
    const uint32_t k = sp_key(v);
    if (k > best) { best = k; at = lo + i; }        // a thread meets its elements in index order
  };
  constexpr int VEC = 16 / sizeof(T);
  if (!((reinterpret_cast<uintptr_t>(x)) & 15)) {
    const int nv = n / VEC;
#pragma unroll 4
    for (int i = tid; i < nv; i += SP_THREADS) {
      const uint4 r = __ldg(reinterpret_cast<const uint4*>(x) + i);
      if constexpr (sizeof(T) == 4) {
        take(4 * i, __uint_as_float(r.x)); take(4 * i + 1, __uint_as_float(r.y)); take(4 * i + 2, __uint_as_float(r.z)); take(4 * i + 3, __uint_as_float(r.w));
      } else {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = unpack_bf16x2(w[j]);
          take(8 * i + 2 * j, f.x);
          take(8 * i + 2 * j + 1, f.y);
        }
      }
    }
    for (int i = nv * VEC + tid; i < n; i += SP_THREADS) take(i, static_cast<float>(x[i]));
  } else {
#pragma unroll 8
    for (int i = tid; i < n; i += SP_THREADS) take(i, static_cast<float>(x[i]));
  }
  // larger key first, then the lower index
  unsigned long long top = (static_cast<unsigned long long>(best) << 32) | (0xFFFFFFFFu - at);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) s.red[warp] = top;
  __syncthreads();
  if (warp == 0) {
    top = lane < SP_WARPS ? s.red[lane] : 0ull;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    top = __shfl_sync(0xffffffffu, top, 0);
  }
  cluster.barrier_wait(std::move(started));
  if (warp == 0) {
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

  // ---- weights: 2^-y with y = (max - x) log2(e) / T = a + i / 256 + r
  const double c = 1.4426950408889634 / static_cast<double>(T_), mxd = mx;
  const float cf = static_cast<float>(c);
  auto weight = [&](float v) -> unsigned long long {
    if (v == mx) return 1ull << SP_ONE;
    const float yf = (mx - v) * cf;
    if (!(yf < SP_ONE + 1.f)) return 0ull;
    const double y = (mxd - static_cast<double>(v)) * c;
    const double big = 6755399441055744.0 / SP_TAB; // 1.5 * 2^52 / 256: adding it leaves round(256 y) in the low bits
    const double z = y + big;
    const int q = __double2loint(z);
    const double r = y - (z - big);                 // |r| <= 2^-9; 2^-r = 1 - z + z^2 / 2 - z^3 / 6, z = r ln 2, to 2e-13
    const double e = fma(r, fma(r, fma(r, -0.055504108664821580, 0.24022650695910071), -0.69314718055994531), 1.0);
    const double f = fma(s.tab[q & (SP_TAB - 1)], e, 4503599627370496.0);       // 2^52: the low bits are the rounded integer
    return (static_cast<unsigned long long>(__double_as_longlong(f)) & 0xFFFFFFFFFFFFFull) >> (q / SP_TAB);
  };

  // ---- the cut: kept are keys above cut_key, and those equal to it with an index up to cut_idx
  uint32_t cut_key = 0;
  int cut_idx = INT_MAX;
  auto cut = [&](uint32_t key, int idx) {
    if (key > cut_key || (key == cut_key && idx < cut_idx)) { cut_key = key; cut_idx = idx; }
  };
  if (min_p > 0.f) {
    const double thr = mxd + static_cast<double>(T_) * log(static_cast<double>(min_p));
    float f = static_cast<float>(thr);
    uint32_t k = sp_key(f + 0.f);
    if (static_cast<double>(f) < thr) ++k;          // the least float that is not below
    cut(k, INT_MAX);
  }
  bool by_k = top_k > 0 && top_k < p.V, by_p = top_p > 0.f && top_p < 1.f;
  if (by_k || by_p) {
    unsigned long long limit = 0, mass_before = 0;  // largest prefix sum; what lies in front of the present subset
    unsigned long long cnt_before = 0;
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
      for (int i = tid; i < SP_BINS; i += SP_THREADS) s.a.h.cnt[i] = s.a.h.lo[i] = s.a.h.hi[i] = 0;
      __syncthreads();
      for (int i = w0 + lane; i < w1; i += 32) {
        const float v = sx[i];
        const int b = bin_of(v);
        if (b < 0) continue;
        atomicAdd(&s.a.h.cnt[b], 1u);
        if (by_p) {
          const unsigned long long w = weight(v);
          const uint32_t l = static_cast<uint32_t>(w), old = atomicAdd(&s.a.h.lo[b], l);
          const uint32_t hi = static_cast<uint32_t>(w >> 32) + (old + l < old ? 1u : 0u);
          if (hi) atomicAdd(&s.a.h.hi[b], hi);
        }
      }
      cluster.sync();
      {                                             // each CTA adds up its share of the bins and tells everyone
        const int share = SP_BINS / C;
        for (int i = tid; i < share; i += SP_THREADS) {
          const int b = rank * share + i;
          uint32_t cnt = 0;
          unsigned long long mass = 0;
          for (int q = 0; q < C; ++q) {
            const SampleShared* r = cluster.map_shared_rank(&s, q);
            cnt += r->a.h.cnt[b];
            mass += (static_cast<unsigned long long>(r->a.h.hi[b]) << 32) + r->a.h.lo[b];
          }
          for (int q = 0; q < C; ++q) {
            SampleShared* r = cluster.map_shared_rank(&s, q);
            r->b.h.cnt[b] = cnt;
            r->b.h.mass[b] = mass;
          }
        }
      }
      if (tid == 0) { s.found = SP_BINS; s.found2 = SP_BINS; s.ncand = 0; }
      cluster.sync();
      // one bin per thread: prefix sums, the first bin in which a limit is passed
      const uint32_t cnt_b = s.b.h.cnt[tid];
      const unsigned long long mass_b = s.b.h.mass[tid];
      unsigned long long cs = warp_scan64(cnt_b), ms = warp_scan64(mass_b);
      if (lane == 31) { s.red[warp] = cs; s.red2[warp] = ms; }
      __syncthreads();
      unsigned long long total = 0;
      for (int w = 0; w < SP_WARPS; ++w) {
        if (w < warp) { cs += s.red[w]; ms += s.red2[w]; }
        total += s.red2[w];
      }
      cs += cnt_before;
      ms += mass_before;
      if (first) limit = static_cast<unsigned long long>(static_cast<double>(top_p) * static_cast<double>(total));
      if (by_k && cs >= static_cast<unsigned long long>(top_k)) atomicMin(&s.found, tid);
      if (by_p && ms > limit) atomicMin(&s.found2, tid);
      __syncthreads();
      const int bk = s.found, bp = s.found2, hit = min(bk, bp);
      if (hit == SP_BINS) break;                    // the rest passes no limit (the same in all CTAs)
      by_k = by_k && bk == hit;
      by_p = by_p && bp == hit;
      if (tid == hit) { s.before[0] = cs - cnt_b; s.before[1] = ms - mass_b; }
      const uint32_t cand = s.b.h.cnt[hit];
      __syncthreads();
      cnt_before = s.before[0];
      mass_before = s.before[1];
      if (cand <= SP_CAND) {
        // ---- rank the candidates
        for (int i = w0 + lane; i < w1; i += 32)
          if (bin_of(sx[i]) == hit) {
            const uint32_t at2 = atomicAdd(&s.ncand, 1u);
            s.a.c.key[at2] = sp_key(sx[i]);
            s.a.c.idx[at2] = lo + i;
          }
        cluster.sync();
        uint32_t mykey[2], myidx[2];
        int have = 0;
        for (int i = tid; i < static_cast<int>(cand); i += SP_THREADS) {        // the i-th of all lists together
          uint32_t j = i;
          int q = 0;
          for (; q < C; ++q) {
            const uint32_t m = cluster.map_shared_rank(&s, q)->ncand;
            if (j < m) break;
            j -= m;
          }
          const SampleShared* r = cluster.map_shared_rank(&s, q);
          mykey[have] = r->a.c.key[j];
          myidx[have++] = r->a.c.idx[j];
        }
        cluster.sync();                             // everyone has read the lists: they become one here
        have = 0;
        for (int i = tid; i < static_cast<int>(cand); i += SP_THREADS) {
          s.a.c.key[i] = mykey[have];
          s.a.c.idx[i] = myidx[have++];
        }
        __syncthreads();
        for (int i = tid; i < static_cast<int>(cand); i += SP_THREADS) {
          const uint32_t k = s.a.c.key[i], d = s.a.c.idx[i];
          int r = 0;
          for (int j = 0; j < static_cast<int>(cand); ++j) r += s.a.c.key[j] > k || (s.a.c.key[j] == k && s.a.c.idx[j] < d);
          s.b.sorted[r] = (static_cast<unsigned long long>(k) << 32) | d;
        }
        __syncthreads();
        if (by_k) cut(static_cast<uint32_t>(s.b.sorted[top_k - cnt_before - 1] >> 32), INT_MAX);
        if (by_p) {                                 // two neighbouring candidates per thread
          unsigned long long w[2], run;
#pragma unroll
          for (int j = 0; j < 2; ++j) w[j] = 2 * tid + j < static_cast<int>(cand) ? weight(sp_unkey(static_cast<uint32_t>(s.b.sorted[2 * tid + j] >> 32))) : 0ull;
          run = warp_scan64(w[0] + w[1]);
          if (lane == 31) s.red[warp] = run;
          if (tid == 0) s.found = 0;
          __syncthreads();
          run += mass_before - w[0] - w[1];
          for (int q = 0; q < warp; ++q) run += s.red[q];
          int keep = 0;
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            run += w[j];
            if (2 * tid + j < static_cast<int>(cand) && run <= limit) keep = 2 * tid + j + 1;
          }
          if (keep) atomicMax(&s.found, keep);
          __syncthreads();
          keep = s.found;
          if (keep == 0 && cnt_before == 0) keep = 1;           // the most probable token stays
          if (keep) cut(static_cast<uint32_t>(s.b.sorted[keep - 1] >> 32), static_cast<int>(static_cast<uint32_t>(s.b.sorted[keep - 1])));
          else cut(static_cast<uint32_t>(s.b.sorted[0] >> 32), static_cast<int>(static_cast<uint32_t>(s.b.sorted[0])) - 1);
        }
        break;
      }
      // ---- too many: divide the bin by the bits of its keys
      uint32_t a = 0xFFFFFFFFu, z = 0;
      for (int i = w0 + lane; i < w1; i += 32)
        if (bin_of(sx[i]) == hit) {
          a = min(a, sp_key(sx[i]));
          z = max(z, sp_key(sx[i]));
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
      unsigned long long keep = cand;
      if (by_p && w) keep = limit > mass_before ? min(keep, (limit - mass_before) / w) : 0ull;
      if (keep == 0 && cnt_before == 0) keep = 1;
      cut(kmin, keep == 0 ? -1 : INT_MAX);
      if (keep && keep < cand) {                    // the index of the last one that stays
        uint32_t mine = 0;
        for (int i = w0 + lane; i < w1; i += 32) mine += sp_key(sx[i]) == kmin;
        mine = __reduce_add_sync(0xffffffffu, mine);
        if (lane == 0) s.red[warp] = mine;
        __syncthreads();
        if (tid < C) {
          unsigned long long m = 0;
          for (int q = 0; q < SP_WARPS; ++q) m += s.red[q];
          cluster.map_shared_rank(&s, tid)->xa[phase][rank] = static_cast<uint32_t>(m);
        }
        cluster.sync();
        unsigned long long left = keep;             // ties up to and with the last one, from this warp's first on
        bool here = true;
        for (int q = 0; q < rank; ++q) { here = here && left > s.xa[phase][q]; left -= s.xa[phase][q]; }
        for (int q = 0; q < warp; ++q) { here = here && left > s.red[q]; left -= s.red[q]; }
        if (here && left <= mine) {
          for (int i0 = w0; i0 < w1; i0 += 32) {
            const bool eq = i0 + lane < w1 && sp_key(sx[i0 + lane]) == kmin;
            const uint32_t vote = __ballot_sync(0xffffffffu, eq);
            const uint32_t m = __popc(vote);
            if (left <= m) {
              if (eq && __popc(vote & ((2u << lane) - 1)) == static_cast<int>(left))
                for (int q = 0; q < C; ++q) cluster.map_shared_rank(&s, q)->xb[phase][0] = lo + i0 + lane;
              break;
            }
            left -= m;
          }
        }
        cluster.sync();
        cut(kmin, static_cast<int>(s.xb[phase][0]));
        phase ^= 1;
      }
      break;
    }
  }

  // ---- sums of the kept weights in index order
  auto kept = [&](int i) -> unsigned long long {
    const uint32_t k = sp_key(sx[i]);
    return k > cut_key || (k == cut_key && lo + i <= cut_idx) ? weight(sx[i]) : 0ull;
  };
  __syncthreads();
  unsigned long long mine = 0;
  for (int i = w0 + lane; i < w1; i += 32) mine += kept(i);
  mine = warp_sum64(mine);
  if (lane == 0) s.red[warp] = mine;
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
  if (front > target || target >= front + mine) return;
  for (int i0 = w0; i0 < w1; i0 += 32) {            // one warp of the row: walk its part
    const unsigned long long run = front + warp_scan64(i0 + lane < w1 ? kept(i0 + lane) : 0ull);
    const uint32_t vote = __ballot_sync(0xffffffffu, run > target);
    if (vote) {
      if (lane == __ffs(vote) - 1) p.out[row] = lo + i0 + lane;
      return;
    }
    front = __shfl_sync(0xffffffffu, run, 31);
  }
}

}  // namespace b200

using namespace b200;

// logits: [B, V] (pitch ld elements), bf16 or fp32; uniform: [B]; per-row tensors may be null (then t, k, p, m hold); out: int64 [B].
B200_API int b200_sample(const SampleParams* a, int B, int is_bf16, void* stream) {
  SampleParams p = *a;
  if (B <= 0 || p.V <= 0 || p.ld < p.V || !p.logits || !p.uniform || !p.out) return -1;
  int C = 1;
  while (C < SP_MAX_CTAS && ((p.V + C - 1) / C > 8192 || (static_cast<long long>(B) * C < 296 && (p.V + C - 1) / C > 1024))) C *= 2;
  p.per = ((p.V + C - 1) / C + SP_THREADS - 1) / SP_THREADS * SP_THREADS;
  const int smem = p.per * 4;
  if (smem > 160 * 1024 || static_cast<long long>(B) * C > (1ll << 31) - 1) return -2;
  auto kern = is_bf16 ? sample_kernel<__nv_bfloat16> : sample_kernel<float>;
  int dev = 0;
  static int configured[64][2] = {};
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -3;
  if (configured[dev][is_bf16 != 0] < smem) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return -4;
    configured[dev][is_bf16 != 0] = smem;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(B * C));
  cfg.blockDim = dim3(SP_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = C;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = g_b200_pdl ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kern, p) == cudaSuccess ? 0 : -10;
}
