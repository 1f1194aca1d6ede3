// Attention of a few query tokens per sequence over the 8-bit cache (kv8.cuh): decode steps, drafted tokens.
//
//   o_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = exp(scale q_i k_j),  j < len - (n - 1 - i)
//
// The rows of a key head (its query heads x the call's tokens) meet every key of the head once, so the kernel is a stream of codes,
// D + D bytes per key, and everything else has to hide behind it.  A warp takes 32 keys at a time through a ring of its own (cp.async, no
// barriers between warps) and forms both products transposed, S^T = K Q^T and O^T = V^T P^T, with mma.sync m16n8k16 on f16: the
// keys (the channels of V) fill the 16 rows, eight query rows the columns.  f16 holds every e4m3 value exactly, and each code is
// widened once.  Transposing matrix loads of bytes turn V.  (mma.sync on 8-bit types was tried first and
// took more instructions per step than widening.  tcgen05 takes codes as they are, but then q and the weights
// have to be split into 8-bit parts, four products each, and a tile's maximum and weights go through barriers of the whole CTA.)
//
// q enters as f16 under a power of two per row, which keeps bf16's eight bits down to 2^-28 of the row's largest.  Weights enter as f16
// times 2^12, and the reference moves only when a score exceeds it by more than 3 (log2 units; most steps of short shares would move
// it otherwise): eleven significant bits for every contribution down to 2^-26 of the largest.
//
// Scales are powers of two: K's enters the score, V's the exponent of the weight, so that the running reference R = max(s + e_v)
// belongs to the contributions to O.  The sum of the weights counts from the middle of the exponents' range, E = 40:
//   O = sum 2^(s + e_v - R) code_v,  l = sum 2^(s + e_v - R) 2^(E - e_v),  o = O / l * 2^E,
// so that its terms stay below 2^95 and none that counts is lost below 2^-126, however far apart the exponents of two blocks are.
// Scores, references, sums and accumulators are fp32.
//
// Work is split evenly whatever the lengths are: the keys of all (sequence, key head, row tile) ranges lie one behind the other in steps of 32,
// and every warp of the machine takes an equal share of them (found from the lengths on the device).  A range that lies in one
// share is written by its warp; one that several warps share leaves partial results that a second kernel joins in their order.
// (Shares of whole CTAs, whose warps met in shared memory at the end of every range, cost 4 us per range of a share, most of it
// the wait for the slowest warp.)
//
// Measured with the joining kernel: 32 sequences of 4096 keys, 32 heads of 96 keep 6.6 TB/s (6.5 with dim 64, 6.3 to 6.7 with 128).  8 sequences of
// 2001 to 4001 keys, 55 heads of 96: 44.5 us, 5.7 TB/s; 65501 and shorter keys, 8 heads of 128 for 32: 41.3 us, 5.0 TB/s, of which finding the
// shares and the first codes take 4 and joining 4.5.  Five drafted tokens, 16 sequences of up to 6007 keys, 8 heads of 64 for 32: 29.7 us; with
// 20 rows a step is 565 instructions, in chains that eight warps to an SM do not cover (40 % of the issue slots).  Issuing a step's score products
// beside the weights of the step before did not help (30.7).  Short ranges are left whole, one to a CTA:
// 512 keys of one sequence, 55 heads of 96: 6.6 us, all latency (7.2 divided and joined by a second kernel).
#include <algorithm>
#include <type_traits>

#include "kv8.cuh"
#include "softmax_math.cuh"

namespace b200 {

struct Kv8Attn {
  const uint8_t *k, *v;
  const int8_t *ke, *ve;
  long long sb, sh, eb, eh;
  int B, Hkv, cap, D, log2_block;
  const __nv_bfloat16* q;            // [B, n, H, D]
  long long q_sb, q_sn, q_sh;
  const int* lens;
  __nv_bfloat16* out;                // [B, n, H, D] contiguous
  float* part;                       // [warps][2][rows][D + 4]: accumulators, reference, sum
  int n, group, rows, tiles_r;       // query tokens, heads per key head, rows per row tile, row tiles
  int most;                          // no length counts for more
  float scale_log2;
  int ctas;
  uint32_t group_magic;              // ceil(2^32 / group)
  int whole;                         // ranges are not divided between shares: each counts as one step of one, a warp's (1) or a CTA's (KA_WARPS)
};

constexpr int KA_WARPS = 4, KA_STEP = 32;           // keys per warp and step
constexpr int KA_MID = 40;                          // E above
constexpr float KA_UP = 12.f, KA_SLACK = 3.f;       // weights reach 2^15
constexpr float KA_NEG = -1.5e38f;                  // "no key yet": finite, so that differences stay defined

// c += a b, a f16 [16 x 16], b f16 [16 x 8]
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Codes of a 16 x 32 operand -> its two 16 x 16 halves in f16: of four neighbouring columns of a lane the first half takes
// the codes of a[0] and a[1], the second those of a[2] and a[3].
__device__ __forceinline__ void widen(const uint32_t (&a)[4], uint32_t (&h)[2][4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    h[i][0] = kv8_half2(a[2 * i], false);
    h[i][1] = kv8_half2(a[2 * i + 1], false);
    h[i][2] = kv8_half2(a[2 * i], true);
    h[i][3] = kv8_half2(a[2 * i + 1], true);
  }
}
// 16 rows x 32 bytes: a[0], a[1] rows g, g + 8 and bytes 4t .. of the first half, a[2], a[3] of the second; 32 rows x 16 bytes, transposed, likewise
__device__ __forceinline__ void ldmatrix4(uint32_t (&a)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix2_trans8(uint32_t (&a)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m16n16.x2.trans.shared.b8 {%0,%1,%2,%3}, [%4];" : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Token of a row (row / group for rows up to 2^32 / group).
__device__ __forceinline__ int kv8_token(const Kv8Attn& p, int row) { return p.group == 1 ? row : static_cast<int>(__umulhi(row, p.group_magic)); }

// Where the steps of every sequence lie and which warp takes which of them (the first total % G take one more than the others); the
// same arithmetic in both kernels.  Every warp holds the lengths of 32 sequences, one per lane.
struct Shares {
  uint32_t total, per_unit;                         // steps; ranges per sequence
  uint32_t G, each, more;                           // warps, steps of each, how many have one more
  int chunk, len;
  __device__ __forceinline__ void load(const Kv8Attn& p, int c) {
    chunk = c;
    const int b = c + (threadIdx.x & 31);
    len = b < p.B ? min(max(__ldg(p.lens + b), 0), p.most) : 0;
  }
  // of a range; without keys it has an empty one
  __device__ __forceinline__ static uint32_t steps(const Kv8Attn& p, int n) { return p.whole ? 1 : max(1, (n + KA_STEP - 1) / KA_STEP); }
  __device__ __forceinline__ uint32_t mine(const Kv8Attn& p) const { return chunk + static_cast<int>(threadIdx.x & 31) < p.B ? steps(p, len) : 0u; }
  __device__ __forceinline__ Shares(const Kv8Attn& p) : total(0), per_unit(p.Hkv * p.tiles_r) {
    for (int c = 0; c < p.B; c += 32) {
      load(p, c);
      total += __reduce_add_sync(0xffffffffu, mine(p));
    }
    total *= per_unit;
    G = min(static_cast<uint32_t>(p.whole == KA_WARPS ? p.ctas : KA_WARPS * p.ctas), total);
    each = total / G;
    more = total - each * G;
  }
  __device__ __forceinline__ uint32_t begin(uint32_t w) const { return w * each + min(w, more); }     // first step of warp w
  __device__ __forceinline__ uint32_t owner(uint32_t step) const {
    const uint32_t wide = more * (each + 1);
    return step < wide ? step / (each + 1) : more + (step - wide) / each;
  }
  __device__ __forceinline__ int length(const Kv8Attn& p, int b) {
    if ((b & ~31) != chunk) load(p, b & ~31);
    return __shfl_sync(0xffffffffu, len, b & 31);
  }
  // The sequence that step `at` belongs to, and its first step.
  __device__ __forceinline__ int find(const Kv8Attn& p, uint32_t at, uint32_t& first) {
    uint32_t before = 0;
    for (int c = 0;; c += 32) {
      if (c != chunk) load(p, c);
      const uint32_t n = mine(p) * per_unit;
      uint32_t sum = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t up = __shfl_up_sync(0xffffffffu, sum, o);
        if ((threadIdx.x & 31) >= o) sum += up;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, before + sum > at);
      if (past || c + 32 >= p.B) {
        const int lane = past ? __ffs(past) - 1 : 0;
        first = before + __shfl_sync(0xffffffffu, sum - n, lane);
        return min(c + lane, p.B - 1);
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  __device__ __forceinline__ uint32_t base(const Kv8Attn& p, int b) {                // first step of sequence b
    uint32_t s = 0;
    for (int c = 0; c <= b; c += 32) {
      if (c != chunk) load(p, c);
      s += __reduce_add_sync(0xffffffffu, c + static_cast<int>(threadIdx.x & 31) < b ? mine(p) : 0u);
    }
    return s * per_unit;
  }
};

// One range after the other of a warp's share.
struct Range {
  int b;
  uint32_t base, step;                              // first step of the sequence; first one that has not been handed out
  int h, r0, len, key0, key1;
  bool begins, ends;                                // the range begins (ends) in this share
  __device__ __forceinline__ void next(const Kv8Attn& p, Shares& sh, uint32_t hi) {
    len = sh.length(p, b);
    uint32_t n = Shares::steps(p, len);
    if (step >= base + n * sh.per_unit) {
      base += n * sh.per_unit;
      len = sh.length(p, ++b);
      n = Shares::steps(p, len);
    }
    const uint32_t unit = (step - base) / n, s0 = (step - base) - unit * n, s1 = min(n, s0 + (hi - step));
    step += s1 - s0;
    h = p.tiles_r == 1 ? unit : unit / static_cast<uint32_t>(p.tiles_r);
    r0 = (unit - h * p.tiles_r) * p.rows;
    if (p.whole) {                                  // the CTA's warps divide the range's steps
      const uint32_t all = max(1, (len + KA_STEP - 1) / KA_STEP), w = p.whole == 1 ? 0 : threadIdx.x >> 5;
      key0 = all * w / p.whole * KA_STEP;
      key1 = min(static_cast<uint32_t>(len), all * (w + 1) / p.whole * KA_STEP);
    } else {
      key0 = s0 * KA_STEP;
      key1 = min(static_cast<uint32_t>(len), s1 * KA_STEP);
    }
    begins = s0 == 0;
    ends = s1 == n;
  }
};

// A warp's ring: stages of 32 K rows and 32 V rows as they lie in the cache, the 16-byte pieces of every 128 bytes exchanged so that no
// eight that a matrix load takes together (K: rows 0, 1, 4, 5, 8, 9, 12, 13 + 2 i; V: eight neighbours) meet in a bank.  (Rows set 16 bytes
// apart would do that, too, but then 128 bytes of a copy fall into more than one line of shared memory: 5.7 instead of 7.0 TB/s.)
template <int D, int NT>
struct Kv8Ring {
  static constexpr int STAGES = D == 128 ? (NT == 1 ? 3 : 2) : D == 96 ? 2 : 3;
  static constexpr int TILE = KA_STEP * D, STAGE = 2 * TILE;
  __device__ __forceinline__ static uint32_t twist(int key) {       // exclusive-ored with the places of a row's pieces (bytes)
    if constexpr (D == 128) return 16 * ((key & 7) ^ ((key >> 2) & 2));
    else if constexpr (D == 64) return 16 * (((key >> 1) & 2) | (((key >> 1) ^ (key >> 3)) & 1));
    else return 16 * (((key >> 2) & 1) | ((key >> 1) & 4));
  }
};

template <int D, int NT>
__host__ __device__ constexpr int kv8_warp_bytes() {        // shared memory of a warp
  return Kv8Ring<D, NT>::STAGES * Kv8Ring<D, NT>::STAGE + (NT > 1 ? NT * (D / 32) * 32 * 16 + 8 * NT * 4 : 0) + 4 * D;
}

// TOGETHER: a range belongs to a CTA, whose warps divide its steps and join their parts.
template <int D, int NT, bool TOGETHER>
__global__ void __launch_bounds__(32 * KA_WARPS, NT > 1 || D == 128 ? 2 : 3)
kv8_attention_kernel(const Kv8Attn p) {
  using Ring = Kv8Ring<D, NT>;
  constexpr int ST = Ring::STAGES, KS = D / 32, VB = D / 16;                 // steps of the score product, blocks of 16 channels
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  // A lane's places: 16-byte pieces of a tile's copy; rows of the matrix loads.  Row r of a score tile is key 4 (r / 2) + r % 2 (+ 2 for
  // r >= 8), so that the weights' pairs are neighbours in V's natural order.
  uint32_t put[VB];
#pragma unroll
  for (int i = 0; i < VB; ++i) put[i] = (16 * (lane + 32 * i)) ^ Ring::twist((lane + 32 * i) / VB);
  const int k_key = 4 * ((lane & 7) >> 1) + (lane & 1) + 2 * ((lane >> 3) & 1);
  const uint32_t k_row = k_key * D + 16 * (lane >> 4), k_twist = Ring::twist(k_key), v_row = lane * D, v_twist = Ring::twist(lane);
  pdl_wait();
  pdl_trigger();                                    // behind the wait: the joining kernel may read the lengths at once
  extern __shared__ __align__(16) uint8_t smem[];   // per warp: ring; (NT > 1) q's fragments, factors of its scores; NaNs noted
  Shares sh(p);
  const uint32_t worker = TOGETHER ? blockIdx.x : warp * p.ctas + blockIdx.x;         // few shares go to different SMs
  if (worker >= sh.G) return;
  const uint32_t hi = sh.begin(worker + 1);
  Range now, nxt;
  nxt.step = sh.begin(worker);
  nxt.b = sh.find(p, nxt.step, nxt.base);

  uint8_t* mem = smem + warp * kv8_warp_bytes<D, NT>();
  uint4* sm_q = reinterpret_cast<uint4*>(mem + ST * Ring::STAGE);
  float* sm_f = reinterpret_cast<float*>(sm_q + (NT > 1 ? NT * KS * 32 : 0));
  int* nan_key = reinterpret_cast<int*>(sm_f + (NT > 1 ? 8 * NT : 0));         // [D] first key with a NaN in this channel, among keys that only some rows see
  const uint32_t ring = smem_u32(mem);

  // Requests run ahead of the products, over the borders of ranges (of which some may be empty).
  Range ahead;
  ahead.b = nxt.b;
  ahead.base = nxt.base;
  ahead.step = nxt.step;
  int ask = 0, ask_end = 0;
  const long long to_v = p.v - p.k;
  const uint8_t* kp = nullptr;                      // this lane's first piece of the step that is requested next
  auto request = [&](int stage) {                   // a step's codes; rows past the end become zero
    while (ask >= ask_end && ahead.step < hi) {
      ahead.next(p, sh, hi);
      ask = ahead.key0;
      ask_end = ahead.key1;
      kp = p.k + ahead.b * p.sb + ahead.h * p.sh + static_cast<long long>(ask) * D + 16 * lane;
    }
    if (ask < ask_end) {
      const uint32_t dst = ring + stage * Ring::STAGE;
      if (ask + KA_STEP <= ask_end) {
#pragma unroll
        for (int i = 0; i < VB; ++i) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + put[i]), "l"(kp + 512 * i) : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + Ring::TILE + put[i]), "l"(kp + to_v + 512 * i) : "memory");
        }
      } else {
        const int left = (ask_end - ask) * D - 16 * lane;
#pragma unroll
        for (int i = 0; i < VB; ++i) {
          const int size = 512 * i < left ? 16 : 0;
          const uint8_t* ks = size ? kp + 512 * i : p.k;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + put[i]), "l"(ks), "r"(size) : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + Ring::TILE + put[i]), "l"(ks + to_v), "r"(size) : "memory");
        }
      }
      kp += KA_STEP * D;
      ask += KA_STEP;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // What a range begins with is loaded while the one before it is worked on: q rows (lane g: row g of a column tile), exponents of the first
  // step.
  uint2 q_raw[NT == 1 ? 2 * KS : 1];
  int kex[2] = {0, 0}, vex[2] = {0, 0};
  auto exponents = [&](const Range& r, int at) {
    const int8_t *kep = p.ke + r.b * p.eb + r.h * p.eh, *vep = p.ve + r.b * p.eb + r.h * p.eh;
    const int e0 = min(at, r.key1 - 1) >> p.log2_block, e1 = min(at + 16, r.key1 - 1) >> p.log2_block;
    kex[0] = __ldg(kep + e0);
    kex[1] = __ldg(kep + e1);
    vex[0] = __ldg(vep + e0);
    vex[1] = __ldg(vep + e1);
  };
  auto q_load = [&](const Range& r, int c8, uint2* raw) {
    const int x = r.r0 + 8 * c8 + g;
    const bool real = 8 * c8 + g < min(p.rows, p.n * p.group - r.r0);
    const int i = real && p.n > 1 ? kv8_token(p, x) : 0, hq = r.h * p.group + (real ? x - i * p.group : 0);
    const __nv_bfloat16* qp = p.q + r.b * p.q_sb + i * p.q_sn + hq * p.q_sh + 4 * t;
#pragma unroll
    for (int j = 0; j < 2 * KS; ++j) raw[j] = real ? __ldg(reinterpret_cast<const uint2*>(qp + 16 * j)) : make_uint2(0u, 0u);
  };
  // f16 fragments of a column tile; returns the factor of its scores, row g
  auto q_convert = [&](const uint2* raw, uint4* to, int pitch) {
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < 2 * KS; ++j) {
      const float2 a = unpack_bf16x2(raw[j].x), c = unpack_bf16x2(raw[j].y);
      amax = fmaxf(fmaxf(fmaxf(amax, kv8_mag(a.x)), kv8_mag(a.y)), fmaxf(kv8_mag(c.x), kv8_mag(c.y)));
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const int e = amax > 0.f ? max((__float_as_int(amax) >> 23) - 127 - 14, -112) : 0;        // largest magnitude in [2^14, 2^15)
    const float f = pow2i(-e);
#pragma unroll
    for (int j = 0; j < KS; ++j) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float2 a = unpack_bf16x2(raw[2 * j + i].x), c = unpack_bf16x2(raw[2 * j + i].y);
        w[2 * i] = half2_bits(a.x * f, a.y * f);
        w[2 * i + 1] = half2_bits(c.x * f, c.y * f);
      }
      to[j * pitch] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return pow2i(e) * p.scale_log2;
  };
  int first_e[4];
  auto prepare = [&](const Range& r) {
    if constexpr (NT == 1) q_load(r, 0, q_raw);
    if (r.key1 > r.key0) {
      const int8_t *kep = p.ke + r.b * p.eb + r.h * p.eh, *vep = p.ve + r.b * p.eb + r.h * p.eh;
      const int e0 = r.key0 >> p.log2_block, e1 = min(r.key0 + 16, r.key1 - 1) >> p.log2_block;
      first_e[0] = __ldg(kep + e0);
      first_e[1] = __ldg(kep + e1);
      first_e[2] = __ldg(vep + e0);
      first_e[3] = __ldg(vep + e1);
    }
  };
  nxt.next(p, sh, hi);
  prepare(nxt);                                     // in front of the bulk of the requests
#pragma unroll 1
  for (int i = 0; i < ST - 1; ++i) request(i);
  if (p.n > 1)
    for (int d = lane; d < D; d += 32) nan_key[d] = INT_MAX;
  int stage = 0;
  bool more = true;

  while (more) {
    now = nxt;
    const int r0 = now.r0, len = now.len, key1 = now.key1;
    const int nrows = min(p.rows, p.n * p.group - r0);

    // q's fragments (per step two halves of 16 channels), and the factor of the raw scores of columns 2t, 2t + 1 without K's scale
    uint4 qf[NT == 1 ? KS : 1];
    float colf[NT][2];
    if constexpr (NT == 1) {
      const float f = q_convert(q_raw, qf, 1);
      colf[0][0] = __shfl_sync(0xffffffffu, f, 8 * t);
      colf[0][1] = __shfl_sync(0xffffffffu, f, 8 * t + 4);
    } else {
      __syncwarp();
      uint2 raw[NT][2 * KS];                        // all of them on their way together
#pragma unroll
      for (int c8 = 0; c8 < NT; ++c8) q_load(now, c8, raw[c8]);
#pragma unroll
      for (int c8 = 0; c8 < NT; ++c8) {
        const float f = q_convert(raw[c8], sm_q + c8 * KS * 32 + lane, 32);
        if (t == 0) sm_f[8 * c8 + g] = f;
      }
      __syncwarp();
#pragma unroll
      for (int c8 = 0; c8 < NT; ++c8) {
        colf[c8][0] = sm_f[8 * c8 + 2 * t];
        colf[c8][1] = sm_f[8 * c8 + 2 * t + 1];
      }
    }
    kex[0] = first_e[0]; kex[1] = first_e[1]; vex[0] = first_e[2]; vex[1] = first_e[3];
    int vmax = KV8_EMIN;                            // largest exponent of V so far
    more = nxt.step < hi;
    if (more) {
      nxt.next(p, sh, hi);
      prepare(nxt);
    }
    // keys that this lane's columns see
    int limit[NT][2];
#pragma unroll
    for (int c8 = 0; c8 < NT; ++c8)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        limit[c8][i] = p.n == 1 ? key1 : min(key1, len - (p.n - 1) + min(kv8_token(p, r0 + 8 * c8 + 2 * t + i), p.n - 1));

    bool noted = false;                             // a NaN of V that only some rows see
    float o[VB][NT][4], R[NT][2], l[NT][2];
#pragma unroll
    for (int c8 = 0; c8 < NT; ++c8) {
#pragma unroll
      for (int i = 0; i < 2; ++i) { R[c8][i] = KA_NEG; l[c8][i] = 0.f; }
#pragma unroll
      for (int w = 0; w < VB; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[w][c8][i] = 0.f;
    }

#pragma unroll 1
    for (int key = now.key0; key < key1; key += KA_STEP) {
      asm volatile("cp.async.wait_group %0;" ::"n"(ST - 2) : "memory");
      __syncwarp();                                 // all lanes' pieces are here, and the stage before has been read
      request(stage == 0 ? ST - 1 : stage - 1);
      const uint32_t here = ring + stage * Ring::STAGE;
      stage = stage == ST - 1 ? 0 : stage + 1;
      // ---- scores of 32 keys, log2 units, V's exponent added
      float s[2][NT][4];
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int c8 = 0; c8 < NT; ++c8)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[m][c8][i] = 0.f;
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        uint32_t x[2][4], a[2][2][4];
#pragma unroll
        for (int m = 0; m < 2; ++m) ldmatrix4(x[m], here + 16 * D * m + ((k_row + 32 * j) ^ k_twist));
#pragma unroll
        for (int m = 0; m < 2; ++m) widen(x[m], a[m]);
#pragma unroll
        for (int c8 = 0; c8 < NT; ++c8) {
          uint4 q4;
          if constexpr (NT == 1) q4 = qf[j];
          else q4 = sm_q[(c8 * KS + j) * 32 + lane];
#pragma unroll
          for (int m = 0; m < 2; ++m) mma_f16(s[m][c8], a[m][0][0], a[m][0][1], a[m][0][2], a[m][0][3], q4.x, q4.y);
#pragma unroll
          for (int m = 0; m < 2; ++m) mma_f16(s[m][c8], a[m][1][0], a[m][1][1], a[m][1][2], a[m][1][3], q4.z, q4.w);
        }
      }
      uint32_t v[VB][4];
      if constexpr (NT == 1) {                      // on its way while the weights are formed
#pragma unroll
        for (int w = 0; w < VB; ++w) ldmatrix2_trans8(v[w], here + Ring::TILE + ((v_row + 16 * w) ^ v_twist));
      }
      const float kf[2] = {pow2i(kex[0]), pow2i(kex[1])}, vf[2] = {static_cast<float>(vex[0]), static_cast<float>(vex[1])};
      vmax = max(vmax, max(vex[0], vex[1]));
      const bool apart = vmax - min(vex[0], vex[1]) > 64;       // weights that are no numbers for O may count in l (all lanes alike)
      const float cf[2] = {apart ? 0.f : pow2i(KA_MID - vex[0]), apart ? 0.f : pow2i(KA_MID - vex[1])};
      exponents(now, key + KA_STEP);
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int c8 = 0; c8 < NT; ++c8)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[m][c8][i] = fmaf(s[m][c8][i], colf[c8][i & 1] * kf[m], vf[m]);
      const bool edge = key + KA_STEP > min(key1, len - (p.n - 1));
      if (edge) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int c8 = 0; c8 < NT; ++c8)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (key + 16 * m + 4 * (g >> 1) + (g & 1) + 2 * (i >> 1) >= limit[c8][i & 1]) s[m][c8][i] = -INFINITY;
      }
      // ---- running reference and weights
      uint32_t pb[NT][4];                           // f16 pairs, column g: keys 4t, 4t + 1 | 4t + 2, 4t + 3 | the same + 16
#pragma unroll
      for (int c8 = 0; c8 < NT; ++c8) {
        float mx[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) mx[i] = fmaxf(fmaxf(s[0][c8][i], s[0][c8][i + 2]), fmaxf(s[1][c8][i], s[1][c8][i + 2]));
        if (__any_sync(0xffffffffu, mx[0] > R[c8][0] + KA_SLACK || mx[1] > R[c8][1] + KA_SLACK)) {    // seldom after the first step
#pragma unroll
          for (int x = 4; x < 32; x <<= 1)
#pragma unroll
            for (int i = 0; i < 2; ++i) mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], x));
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float rn = fmaxf(R[c8][i], mx[i]), half = ex2_approx(0.5f * (R[c8][i] - rn)), alpha = half * half;
            R[c8][i] = rn;
            l[c8][i] = l[c8][i] * half * half;      // alpha may be too small for a number where this is not
#pragma unroll
            for (int w = 0; w < VB; ++w) {
              o[w][c8][i] *= alpha;
              o[w][c8][i + 2] *= alpha;
            }
          }
        }
        const float up[2] = {R[c8][0] - KA_UP, R[c8][1] - KA_UP};
        if (apart) {
#pragma unroll
          for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) l[c8][i & 1] += ex2_approx(s[m][c8][i] - up[i & 1] - vf[m] + KA_MID);
        }
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          float w4[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            w4[i] = ex2_approx(s[m][c8][i] - up[i & 1]);
            l[c8][i & 1] = fmaf(w4[i], cf[m], l[c8][i & 1]);
          }
          pb[c8][2 * m] = transpose8x8(half2_bits(w4[0], w4[1]));
          pb[c8][2 * m + 1] = transpose8x8(half2_bits(w4[2], w4[3]));
        }
      }
      // ---- O^T += V^T P^T
      if constexpr (NT > 1) {
#pragma unroll
        for (int w = 0; w < VB; ++w) ldmatrix2_trans8(v[w], here + Ring::TILE + ((v_row + 16 * w) ^ v_twist));
      }
      if (edge && p.n > 1) {                        // weights of zero do not hide a NaN of V: one that only some rows see is noted
#pragma unroll
        for (int w = 0; w < VB; ++w)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t nan = ((v[w][i] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
            if (nan) {
              noted = true;
              for (int y = 0; y < 4; ++y)
                if (nan >> (8 * y + 7) & 1u) {
                  atomicMin(&nan_key[16 * w + g + 8 * (i & 1)], key + 16 * (i >> 1) + 4 * t + y);
                  v[w][i] &= ~(0xFFu << (8 * y));
                }
            }
          }
      }
#pragma unroll
      for (int w = 0; w < VB; ++w) {
        uint32_t x[2][4];
        widen(v[w], x);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int c8 = 0; c8 < NT; ++c8) mma_f16(o[w][c8], x[i][0], x[i][1], x[i][2], x[i][3], pb[c8][2 * i], pb[c8][2 * i + 1]);
      }
    }

    // ---- the range's outputs, or this share's part of them
    const bool whole = now.begins && now.ends && !TOGETHER;
    noted = __any_sync(0xffffffffu, noted);
#pragma unroll
    for (int c8 = 0; c8 < NT; ++c8)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float sum = l[c8][i];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        const int c = 8 * c8 + 2 * t + i;
        if (c < nrows) {
          const int row = r0 + c, tok = p.n == 1 ? 0 : kv8_token(p, row), hq = now.h * p.group + row - tok * p.group;
          if (noted) {
            const int sees = len - (p.n - 1) + tok;
#pragma unroll
            for (int w = 0; w < VB; ++w) {
              if (nan_key[16 * w + g] < sees) o[w][c8][i] = NAN;
              if (nan_key[16 * w + g + 8] < sees) o[w][c8][i + 2] = NAN;
            }
          }
          if (whole) {
            const float f = sum == 0.f ? 0.f : 1.f / sum, e = pow2i(KA_MID);
            __nv_bfloat16* to = p.out + ((static_cast<size_t>(now.b) * p.n + tok) * p.Hkv * p.group + hq) * D + g;
#pragma unroll
            for (int w = 0; w < VB; ++w) {
              to[16 * w] = f2bf(o[w][c8][i] * e * f);
              to[16 * w + 8] = f2bf(o[w][c8][i + 2] * e * f);
            }
          } else {
            float* to = p.part + ((TOGETHER ? static_cast<long long>(KA_WARPS) * worker + warp : 2ll * worker + (now.begins ? 1 : 0)) * p.rows + c) * (D + 4) + g;
#pragma unroll
            for (int w = 0; w < VB; ++w) {
              to[16 * w] = o[w][c8][i];
              to[16 * w + 8] = o[w][c8][i + 2];
            }
            if (g == 0) *reinterpret_cast<float2*>(to + D) = make_float2(R[c8][i], sum);
          }
        }
      }
    if (noted) {
      __syncwarp();
      for (int d = lane; d < D; d += 32) nan_key[d] = INT_MAX;
      __syncwarp();
    }
    if constexpr (TOGETHER) {                       // the warps' parts, by way of L2
      __syncthreads();
      constexpr int AT_ONCE = NT == 1 ? 2 : 4;      // rows whose loads a warp has in flight
#pragma unroll 1
      for (int c0 = warp; c0 < nrows; c0 += AT_ONCE * KA_WARPS) {
        float2 ml[AT_ONCE][KA_WARPS];
        float4 v[AT_ONCE][KA_WARPS];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
          for (int w = 0; w < KA_WARPS; ++w) {
            const int c = min(c0 + KA_WARPS * i, nrows - 1);
            const float* from = p.part + ((static_cast<long long>(KA_WARPS) * worker + w) * p.rows + c) * (D + 4);
            ml[i][w] = *reinterpret_cast<const float2*>(from + D);
            v[i][w] = lane < D / 4 ? *reinterpret_cast<const float4*>(from + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
          }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
          const int c = c0 + KA_WARPS * i;
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
          float top = KA_NEG, sum = 0.f;
#pragma unroll
          for (int w = 0; w < KA_WARPS; ++w) top = fmaxf(top, ml[i][w].x);
#pragma unroll
          for (int w = 0; w < KA_WARPS; ++w) {
            const float half = ex2_approx(0.5f * (ml[i][w].x - top)), f = half * half;
            sum += ml[i][w].y * half * half;
            acc.x = fmaf(v[i][w].x, f, acc.x); acc.y = fmaf(v[i][w].y, f, acc.y); acc.z = fmaf(v[i][w].z, f, acc.z); acc.w = fmaf(v[i][w].w, f, acc.w);
          }
          const int row = r0 + c, tok = p.n == 1 ? 0 : kv8_token(p, row), hq = now.h * p.group + row - tok * p.group;
          const float f = sum == 0.f ? 0.f : 1.f / sum, e = pow2i(KA_MID);
          if (c < nrows && lane < D / 4)
            *reinterpret_cast<uint2*>(p.out + ((static_cast<size_t>(now.b) * p.n + tok) * p.Hkv * p.group + hq) * D + 4 * lane) =
                make_uint2(pack_bf16x2(acc.x * e * f, acc.y * e * f), pack_bf16x2(acc.z * e * f, acc.w * e * f));
        }
      }
      __syncthreads();
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// Joins the partial results of ranges that several warps shared.  WR warps per row of a range take every WR-th part; grid (rows of a
// sequence, B), blocks of at least four warps.  Launched so that it finds its places while the kernel above is still at work.
template <int D, int WR>
__global__ void __launch_bounds__(WR > 4 ? 32 * WR : 128)
kv8_join_kernel(const Kv8Attn p) {
  constexpr int AT_ONCE = 8, WARPS = WR > 4 ? WR : 4;       // parts whose loads a warp has in flight
  __shared__ float4 sm[WARPS][D / 4];
  const int b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, idx = blockIdx.x * (WARPS / WR) + warp / WR, place = warp % WR;
  Shares sh(p);                                     // the lengths were there before the kernel above began
  const uint32_t base = sh.base(p, b), n = Shares::steps(p, sh.length(p, b));
  const int unit = idx / p.rows, r = idx - unit * p.rows;
  const int h = unit / p.tiles_r, row = (unit - h * p.tiles_r) * p.rows + r;
  const bool mine = n > 1 && unit < static_cast<int>(sh.per_unit) && row < p.n * p.group;
  const int c0 = mine ? sh.owner(base + unit * n) : 0, parts = mine ? sh.owner(base + unit * n + n - 1) - c0 + 1 : 1;
  pdl_trigger();
  pdl_wait();
  if (WR >= 4 && parts == 1) return;                // written by its warp
  // the warp that begins the range kept it in its second place, the others in their first
  auto part = [&](int x) { return p.part + ((2ll * (c0 + x) + (x == 0 ? 1 : 0)) * p.rows + r) * (D + 4); };
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float top = KA_NEG, sum = 0.f;
  for (int x0 = 0; x0 < parts && parts > 1; x0 += WR * AT_ONCE) {
    constexpr int ML = (WR * AT_ONCE + 31) / 32;    // references and sums of all parts of the round, a lane each
    float2 ml[ML];
#pragma unroll
    for (int i = 0; i < ML; ++i) {
      const int x = 32 * i + lane;
      ml[i] = x < WR * AT_ONCE && x0 + x < parts ? *reinterpret_cast<const float2*>(part(x0 + x) + D) : make_float2(KA_NEG, 0.f);
    }
    float4 v[AT_ONCE];
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const int x = x0 + WR * i + place;
      v[i] = x < parts && lane < D / 4 ? *reinterpret_cast<const float4*>(part(x) + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float tn = top, s = 0.f;
#pragma unroll
    for (int i = 0; i < ML; ++i) tn = fmaxf(tn, ml[i].x);
    tn = warp_max(tn);
    const float f0h = ex2_approx(0.5f * (top - tn)), f0 = f0h * f0h;
    top = tn;
#pragma unroll
    for (int i = 0; i < ML; ++i) {
      const float half = ex2_approx(0.5f * (ml[i].x - tn));     // twice, as above
      ml[i].x = half * half;
      s += ml[i].y * half * half;
    }
    sum = sum * f0h * f0h + warp_sum(s);
    acc.x *= f0; acc.y *= f0; acc.z *= f0; acc.w *= f0;
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {             // part WR i + place: lane (WR i + place) % 32 of round (WR i + place) / 32
      const float f = __shfl_sync(0xffffffffu, ml[WR * i / 32].x, (WR * i) % 32 + place);
      acc.x = fmaf(v[i].x, f, acc.x); acc.y = fmaf(v[i].y, f, acc.y); acc.z = fmaf(v[i].z, f, acc.z); acc.w = fmaf(v[i].w, f, acc.w);
    }
  }
  if constexpr (WR > 1) {
    if (lane < D / 4) sm[warp][lane] = acc;
    __syncthreads();
    if (place || lane >= D / 4) return;
#pragma unroll
    for (int i = 1; i < WR; ++i) {
      const float4 y = sm[warp + i][lane];
      acc.x += y.x; acc.y += y.y; acc.z += y.z; acc.w += y.w;
    }
  }
  if (parts == 1 || lane >= D / 4) return;
  const float f = sum == 0.f ? 0.f : 1.f / sum, e = pow2i(KA_MID);
  const int i = row / p.group, hq = h * p.group + row - i * p.group;
  *reinterpret_cast<uint2*>(p.out + ((static_cast<size_t>(b) * p.n + i) * p.Hkv * p.group + hq) * D + 4 * lane) =
      make_uint2(pack_bf16x2(acc.x * e * f, acc.y * e * f), pack_bf16x2(acc.z * e * f, acc.w * e * f));
}

template <int D, int NT, bool TOGETHER>
static int kv8_slots() {                            // CTAs that one SM holds
  auto kern = kv8_attention_kernel<D, NT, TOGETHER>;
  constexpr int smem = KA_WARPS * kv8_warp_bytes<D, NT>();
  int dev = 0, per = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  static int known[64] = {};
  if (!known[dev]) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kern, 32 * KA_WARPS, smem) != cudaSuccess || per < 1)
      return 0;
    known[dev] = per;
  }
  return known[dev];
}

template <int D>
static int kv8_slots_d(int nt) {
  switch (nt) {
    case 1: return std::min(kv8_slots<D, 1, false>(), kv8_slots<D, 1, true>());
    case 2: return std::min(kv8_slots<D, 2, false>(), kv8_slots<D, 2, true>());
    case 3: return std::min(kv8_slots<D, 3, false>(), kv8_slots<D, 3, true>());
    case 4: return std::min(kv8_slots<D, 4, false>(), kv8_slots<D, 4, true>());
    default: return 0;
  }
}
static int kv8_slots_any(int D, int nt) {
  switch (D) {
    case 32: return kv8_slots_d<32>(nt);
    case 64: return kv8_slots_d<64>(nt);
    case 96: return kv8_slots_d<96>(nt);
    case 128: return kv8_slots_d<128>(nt);
    default: return 0;
  }
}

template <int D, int WR>
static void kv8_join(const Kv8Attn& p, cudaStream_t st) {
  constexpr int WARPS = WR > 4 ? WR : 4;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((p.Hkv * p.tiles_r * p.rows + WARPS / WR - 1) / (WARPS / WR), p.B);
  cfg.blockDim = dim3(32 * WARPS);
  cfg.stream = st;
  cudaLaunchAttribute at[1];                        // its launch overlaps the kernel whose completion it waits for
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, kv8_join_kernel<D, WR>, p);
}

template <int D>
static void kv8_run(const Kv8Attn& p, int nt, cudaStream_t st) {
  const dim3 block(32 * KA_WARPS), grid(p.ctas);
  auto run = [&](auto columns, auto together) {
    constexpr int NT = decltype(columns)::value;
    launch_k(kv8_attention_kernel<D, NT, decltype(together)::value>, grid, block, KA_WARPS * kv8_warp_bytes<D, NT>(), st, p);
  };
  auto pick = [&](auto together) {
    if (nt == 1) run(std::integral_constant<int, 1>(), together);
    else if (nt == 2) run(std::integral_constant<int, 2>(), together);
    else if (nt == 3) run(std::integral_constant<int, 3>(), together);
    else run(std::integral_constant<int, 4>(), together);
  };
  if (p.whole == KA_WARPS) pick(std::true_type());
  else pick(std::false_type());
  if (p.whole) return;
  // warps per row of a range by the parts that a range has on average, as long as the machine holds them all at a time
  const long long ranges = static_cast<long long>(p.B) * p.Hkv * p.tiles_r, parts = static_cast<long long>(KA_WARPS) * p.ctas / ranges;
  if (parts > 32 && ranges * p.rows <= 256) kv8_join<D, 16>(p, st);
  else if (parts >= 8 && ranges * p.rows <= 1024) kv8_join<D, 4>(p, st);
  else kv8_join<D, 1>(p, st);
}

}  // namespace b200

using namespace b200;

// Ranges of few steps are left whole: the warps of a CTA (KA_WARPS), or where there are more ranges than CTAs a warp (1), go through one of
// them sooner than a second kernel joins its parts, and a launch is saved.  Divided and whole, us: 55 ranges of 256 keys 6.8 and 5.6, of 1024 8.8 and 9.0;
// 440 ranges of 256 keys 7.8 and 6.9, of 1024 14.5 and 12.8; two ranges of sixteen rows and 256 keys 6.9 and 7.1, 512 keys 6.8 and 8.8;
// 1024 ranges of 128 keys 8.7 and (1) 6.7.
static int kv8_whole(long long ranges, int most, long long slots) {
  const int steps = (most + KA_STEP - 1) / KA_STEP;
  return ranges <= slots && steps <= (ranges < 16 ? 12 : 32) ? KA_WARPS : steps <= 6 ? 1 : 0;
}

// How a call is cut.  plan: [0] rows per row tile, [1] row tiles, [2] CTAs, [3] floats of scratch, [4] whole ranges.
B200_API int b200_kv8_attention_plan(int B, int Hkv, int D, int rows, int most, int* plan) {
  if (B <= 0 || B > 65535 || Hkv <= 0 || rows <= 0 || most <= 0) return -1;
  const int tiles_r = (rows + 31) / 32, per = (rows + tiles_r - 1) / tiles_r;
  const int slots = kv8_slots_any(D, (per + 7) / 8);
  if (!slots) return -2;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return -3;
  const long long steps = static_cast<long long>(B) * Hkv * tiles_r * ((static_cast<long long>(most) + KA_STEP - 1) / KA_STEP);
  if (steps > (1ll << 31) - 1 || static_cast<long long>(Hkv) * tiles_r * per > (1ll << 31) - 4) return -4;
  const long long ranges = static_cast<long long>(B) * Hkv * tiles_r, most_ctas = static_cast<long long>(sms) * slots;
  const int whole = kv8_whole(ranges, most, most_ctas);
  plan[0] = per;
  plan[1] = tiles_r;
  plan[2] = static_cast<int>(std::min(whole ? ranges : steps, most_ctas));
  plan[3] = whole == 1 ? 0 : KA_WARPS * plan[2] * (whole ? 1 : 2) * per * (D + 4);
  plan[4] = whole;
  return 0;
}

// a: sizes and cache of the call (rows, tiles_r, ctas, whole and the size of part as planned); the tensors of this call apart from it.
B200_API int b200_kv8_attention(const Kv8Attn* a, const void* q, const int* lens, void* out, float* part, void* stream) {
  Kv8Attn p = *a;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.lens = lens;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.part = part;
  if (p.B <= 0 || p.B > 65535 || p.Hkv <= 0 || p.n <= 0 || p.group <= 0 || p.rows <= 0 || p.rows > 32 || p.tiles_r <= 0 || p.ctas <= 0 ||
      p.log2_block < 4 || p.log2_block > 7 || p.most <= 0 || p.most > p.cap)
    return -1;
  if ((p.whole != 0 && p.whole != 1 && p.whole != KA_WARPS) || (p.whole != 1 && !p.part)) return -1;
  if (static_cast<long long>(p.rows) * p.tiles_r < static_cast<long long>(p.n) * p.group) return -1;
  if (static_cast<double>(p.n) * p.group * p.group > 4e9) return -4;
  p.group_magic = static_cast<uint32_t>((0x100000000ull + p.group - 1) / p.group);
  if ((reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) | p.sb | p.sh) & 15) return -2;
  if (((reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.out) | reinterpret_cast<uintptr_t>(p.part)) & 15) || ((p.q_sb | p.q_sn | p.q_sh) & 7)) return -2;
  const int nt = (p.rows + 7) / 8;
  if (!kv8_slots_any(p.D, nt)) return -3;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  switch (p.D) {
    case 32: kv8_run<32>(p, nt, st); break;
    case 64: kv8_run<64>(p, nt, st); break;
    case 96: kv8_run<96>(p, nt, st); break;
    case 128: kv8_run<128>(p, nt, st); break;
    default: return -1;
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -10;
}
