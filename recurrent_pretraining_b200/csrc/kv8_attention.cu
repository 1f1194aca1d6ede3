// Attention of a few query tokens per sequence over the 8-bit cache (kv8.cuh): decode steps, drafted tokens.
//
//   o_i = sum_j w_ij v_j / sum_j w_ij,  w_ij = exp(scale q_i k_j),  j < len - (n - 1 - i)
//
// The rows of a key head (its query heads x the call's tokens) meet every key of the head once, so the kernel is a stream of codes:
// D + D bytes per key.  Both products are formed transposed, S^T = K Q^T and O^T = V^T P^T, with mma.sync m16n8k16: the keys (the channels
// of V) fill the 16 rows and the query rows the 8 columns, of which a single token of ungrouped heads fills one (a tcgen05 tile would
// hold 128 rows of keys at least, but wants its operands as 16-bit tiles in shared memory: an unpacking pass in front of every product
// that this form does not have).  Codes go from global memory to registers and become f16 there, which holds
// every e4m3 value exactly.  The order of a dot product's terms is free, so a lane takes 8 to 16 neighbouring bytes of a key row as
// they lie in memory and q's fragments follow that order; likewise the rows of V^T.
//
// Scales are powers of two: K's enters the score, V's the exponent of the weight, so that the running reference R = max(s + e_v)
// belongs to the contributions to O.  The sum of the weights counts from e_ref, the exponent of the sequence's first block of values:
//   O = sum 2^(s + e_v - R) code_v,  l = sum 2^(s + e_v - R) 2^(e_ref - e_v),  o = O / l * 2^e_ref.
// Weights enter the product with V as f16 times 2^15: eleven significant bits for every contribution down to 2^-29 of the largest.
// q enters as f16 under a power of two per row, which keeps bf16's eight bits down to 2^-28 of the row's largest.
// Scores, references, sums and accumulators are fp32.
//
// Work is split evenly whatever the lengths are: the (sequence, key head, row tile) ranges lie one behind the other in tiles of keys, and every CTA
// takes an equal share of all tiles (read from the lengths on the device).  A range that several CTAs share leaves partial results
// that a second kernel joins in their order; a range that lies in one CTA is written by it.  Without long sequences a tile is a
// whole range and the second kernel is left out.
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
  float* part;                       // [CTAs][2][rows][D + 2]; null: a tile is a whole range
  int n, group, rows, tiles_r;       // query tokens, heads per key head, rows per row tile, row tiles
  int tile, most;                    // keys per tile (a multiple of 128); no length counts for more than `most`
  float scale_log2;
};

constexpr int KA_WARPS = 4, KA_STEP = 32;           // keys per warp and step
constexpr float KA_NEG = -1.5e38f;                  // "no key yet": finite, so that differences stay defined

__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Where the tiles of every sequence lie and which CTA takes which of them; the same arithmetic in both kernels.
struct Shares {
  long long total;
  int per_unit;                                     // ranges per sequence
  __device__ int tiles_of(const Kv8Attn& p, int b) const {     // per range; a sequence without keys has one empty tile
    const int len = min(max(p.lens[b], 0), p.most);
    return max(1, (len + p.tile - 1) / p.tile);
  }
  __device__ Shares(const Kv8Attn& p) : total(0), per_unit(p.Hkv * p.tiles_r) {
    for (int b = threadIdx.x & 31; b < p.B; b += 32) total += tiles_of(p, b);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    total *= per_unit;
  }
  // The sequence that tile `at` belongs to and its first tile; by the whole warp, 32 sequences at a time.
  __device__ int find(const Kv8Attn& p, long long at, long long& first) const {
    long long before = 0;
    for (int b0 = 0;; b0 += 32) {
      const int b = b0 + (threadIdx.x & 31);
      const long long mine = b < p.B ? static_cast<long long>(tiles_of(p, b)) * per_unit : 0;
      long long sum = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, sum, o);
        if ((threadIdx.x & 31) >= o) sum += up;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, before + sum > at);
      if (past || b0 + 32 >= p.B) {
        const int lane = past ? __ffs(past) - 1 : 0;
        first = before + __shfl_sync(0xffffffffu, sum - mine, lane);
        return min(b0 + lane, p.B - 1);
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  // first tile of sequence b (summed by the whole warp)
  __device__ long long base(const Kv8Attn& p, int b) const {
    long long s = 0;
    for (int i = threadIdx.x & 31; i < b; i += 32) s += tiles_of(p, i);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s * per_unit;
  }
};

template <int D, int NT>
__global__ void __launch_bounds__(32 * KA_WARPS)
kv8_attention_kernel(const Kv8Attn p) {
  constexpr int KW = D / 16;                        // words of a key row per lane = steps of the score product
  constexpr int VW = D / 32;                        // words of a value row per lane
  pdl_trigger();
  pdl_wait();
  extern __shared__ float sm[];                     // [warps][rows][D] accumulators, [warps][rows] references, sums; q fragments (NT > 1)
  __shared__ int nan_key[D];                        // first key with a NaN in this channel, among keys that only some rows see
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float* sm_o = sm;
  float* sm_r = sm + KA_WARPS * p.rows * D;
  float* sm_l = sm_r + KA_WARPS * p.rows;
  uint2* sm_q = reinterpret_cast<uint2*>(sm_l + KA_WARPS * p.rows);
  float* sm_f = reinterpret_cast<float*>(sm_q + NT * KW * 32);
  const Shares sh(p);
  const long long G = min(static_cast<long long>(gridDim.x), sh.total);
  if (blockIdx.x >= G) return;
  const long long lo = blockIdx.x * sh.total / G, hi = (blockIdx.x + 1) * sh.total / G;
  for (int d = threadIdx.x; d < D; d += 32 * KA_WARPS) nan_key[d] = INT_MAX;

  __syncthreads();
  long long base;                                   // first tile of sequence b
  int b = sh.find(p, lo, base);
  // channels of this lane: k-step j of the score product / word w of a value row
  auto k_dim = [&](int j) { return j < 4 * (D / 64) ? 64 * (j / 4) + 16 * t + 4 * (j % 4) : 64 * (D / 64) + 8 * t + 4 * (j - 4 * (D / 64)); };
  auto v_dim = [&](int w) { return D == 128 ? 16 * g + 4 * w : D == 96 ? (w < 2 ? 8 * g + 4 * w : 64 + 4 * g) : D == 64 ? 8 * g + 4 * w : 4 * g; };

  for (long long tile = lo; tile < hi;) {
    int nt = sh.tiles_of(p, b);
    if (tile >= base + static_cast<long long>(nt) * sh.per_unit) {
      base += static_cast<long long>(nt) * sh.per_unit;
      nt = sh.tiles_of(p, ++b);
    }
    const int unit = static_cast<int>(tile - base) / nt, t0 = static_cast<int>(tile - base) - unit * nt;    // a sequence has fewer than 2^31 tiles
    const int t1 = static_cast<int>(min(static_cast<long long>(nt), t0 + (hi - tile)));
    tile += t1 - t0;
    const int h = unit / p.tiles_r, r0 = (unit - h * p.tiles_r) * p.rows;
    const int nrows = min(p.rows, p.n * p.group - r0);
    const int len = min(max(p.lens[b], 0), p.most);
    const int key0 = t0 * p.tile, key1 = min(len, t1 * p.tile);
    const uint8_t* kp = p.k + b * p.sb + h * p.sh;
    const uint8_t* vp = p.v + b * p.sb + h * p.sh;
    const int8_t* kep = p.ke + b * p.eb + h * p.eh;
    const int8_t* vep = p.ve + b * p.eb + h * p.eh;

    uint32_t kr[2][2][KW], vr[2][4][VW];
    int kex[2], vex[2];
    auto load_k = [&](int key) {                    // keys `key` .. + 31 of this warp; rows past the end repeat the last key
#pragma unroll
      for (int m = 0; m < 2; ++m) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint8_t* row = kp + static_cast<long long>(min(key + 16 * m + 8 * r + g, key1 - 1)) * D;
#pragma unroll
          for (int i = 0; i < D / 64; ++i) {
            const uint4 x = __ldg(reinterpret_cast<const uint4*>(row + 64 * i + 16 * t));
            kr[m][r][4 * i] = x.x; kr[m][r][4 * i + 1] = x.y; kr[m][r][4 * i + 2] = x.z; kr[m][r][4 * i + 3] = x.w;
          }
          if constexpr (D % 64 != 0) {
            const uint2 x = __ldg(reinterpret_cast<const uint2*>(row + 64 * (D / 64) + 8 * t));
            kr[m][r][KW - 2] = x.x; kr[m][r][KW - 1] = x.y;
          }
        }
        kex[m] = __ldg(kep + (min(key + 16 * m, key1 - 1) >> p.log2_block));
      }
    };
    auto load_v = [&](int key) {
#pragma unroll
      for (int m = 0; m < 2; ++m) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = key + 16 * m + 2 * t + (i & 1) + 8 * (i >> 1);
          const uint8_t* row = vp + static_cast<long long>(min(at, key1 - 1)) * D;
          if constexpr (D == 128) {
            const uint4 x = __ldg(reinterpret_cast<const uint4*>(row + 16 * g));
            vr[m][i][0] = x.x; vr[m][i][1] = x.y; vr[m][i][2] = x.z; vr[m][i][3] = x.w;
          } else if constexpr (D == 32) {
            vr[m][i][0] = __ldg(reinterpret_cast<const uint32_t*>(row + 4 * g));
          } else {
            const uint2 x = __ldg(reinterpret_cast<const uint2*>(row + 8 * g));
            vr[m][i][0] = x.x; vr[m][i][1] = x.y;
            if constexpr (D == 96) vr[m][i][2] = __ldg(reinterpret_cast<const uint32_t*>(row + 64 + 4 * g));
          }
        }
        vex[m] = __ldg(vep + (min(key + 16 * m, key1 - 1) >> p.log2_block));
      }
    };

    int key = key0 + KA_STEP * warp;
    const bool any = key < key1;
    if (any) { load_k(key); load_v(key); }
    const int e_ref = key1 > key0 ? __ldg(vep) : 0;

    // q of this lane's column (row r0 + 8 nt + g), under a power of two per row
    uint2 qf[NT == 1 ? KW : 1];
    float colf[NT][2];                              // factor of the raw scores of columns 2t, 2t + 1, without K's scale
    auto q_fragments = [&](int c8, auto&& put) {
      const int r = r0 + 8 * c8 + g;
      const bool real = 8 * c8 + g < nrows;
      const int i = real ? r / p.group : 0, hq = h * p.group + (real ? r - i * p.group : 0);
      const __nv_bfloat16* qp = p.q + b * p.q_sb + i * p.q_sn + hq * p.q_sh;
      uint2 raw[KW];
      float amax = 0.f;
#pragma unroll
      for (int j = 0; j < KW; ++j) {
        raw[j] = real ? __ldg(reinterpret_cast<const uint2*>(qp + k_dim(j))) : make_uint2(0u, 0u);
        const float2 a = unpack_bf16x2(raw[j].x), c = unpack_bf16x2(raw[j].y);
        amax = fmaxf(fmaxf(fmaxf(amax, kv8_mag(a.x)), kv8_mag(a.y)), fmaxf(kv8_mag(c.x), kv8_mag(c.y)));
      }
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const int e = amax > 0.f ? max((__float_as_int(amax) >> 23) - 127 - 14, -112) : 0;      // largest magnitude in [2^14, 2^15)
      const float f = pow2i(-e);
#pragma unroll
      for (int j = 0; j < KW; ++j) {
        const float2 a = unpack_bf16x2(raw[j].x), c = unpack_bf16x2(raw[j].y);
        put(j, make_uint2(half2_bits(a.x * f, a.y * f), half2_bits(c.x * f, c.y * f)));
      }
      return pow2i(e) * p.scale_log2;
    };
    if constexpr (NT == 1) {
      const float f = q_fragments(0, [&](int j, uint2 x) { qf[j] = x; });
      colf[0][0] = __shfl_sync(0xffffffffu, f, 8 * t);
      colf[0][1] = __shfl_sync(0xffffffffu, f, 8 * t + 4);
    } else {
      __syncthreads();                              // the previous range's fragments have been used
      for (int c8 = warp; c8 < NT; c8 += KA_WARPS) {
        const float f = q_fragments(c8, [&](int j, uint2 x) { sm_q[(c8 * KW + j) * 32 + lane] = x; });
        if (t == 0) sm_f[8 * c8 + g] = f;
      }
      __syncthreads();
#pragma unroll
      for (int c8 = 0; c8 < NT; ++c8) {
        colf[c8][0] = sm_f[8 * c8 + 2 * t];
        colf[c8][1] = sm_f[8 * c8 + 2 * t + 1];
      }
    }
    // keys that this lane's columns see
    int limit[NT][2];
#pragma unroll
    for (int c8 = 0; c8 < NT; ++c8)
#pragma unroll
      for (int i = 0; i < 2; ++i) limit[c8][i] = len - (p.n - 1) + min((r0 + 8 * c8 + 2 * t + i) / p.group, p.n - 1);

    float o[VW][2][NT][4], R[NT][2], l[NT][2];
#pragma unroll
    for (int c8 = 0; c8 < NT; ++c8) {
#pragma unroll
      for (int i = 0; i < 2; ++i) { R[c8][i] = KA_NEG; l[c8][i] = 0.f; }
#pragma unroll
      for (int w = 0; w < VW; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[w][0][c8][i] = o[w][1][c8][i] = 0.f;
    }

    for (; key < key1; key += KA_STEP * KA_WARPS) {
      // ---- scores of 32 keys, log2 units, V's exponent added
      float s[2][NT][4];
      const bool more = key + KA_STEP * KA_WARPS < key1;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
#pragma unroll
        for (int c8 = 0; c8 < NT; ++c8)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[m][c8][i] = 0.f;
#pragma unroll
        for (int j = 0; j < KW; ++j) {
          const uint32_t a[4] = {kv8_half2(kr[m][0][j], false), kv8_half2(kr[m][1][j], false), kv8_half2(kr[m][0][j], true), kv8_half2(kr[m][1][j], true)};
#pragma unroll
          for (int c8 = 0; c8 < NT; ++c8) {
            uint2 q2;
            if constexpr (NT == 1) q2 = qf[j];
            else q2 = sm_q[(c8 * KW + j) * 32 + lane];
            mma_f16(s[m][c8], a, q2.x, q2.y);
          }
        }
      }
      const float kf[2] = {pow2i(kex[0]), pow2i(kex[1])}, vf[2] = {static_cast<float>(vex[0]), static_cast<float>(vex[1])};
      const float cf[2] = {pow2i(min(e_ref - vex[0], 127)), pow2i(min(e_ref - vex[1], 127))};
      if (more) load_k(key + KA_STEP * KA_WARPS);
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int c8 = 0; c8 < NT; ++c8)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[m][c8][i] = fmaf(s[m][c8][i], colf[c8][i & 1] * kf[m], vf[m]);
      const bool edge = key + KA_STEP > len - (p.n - 1) || key + KA_STEP > key1;
      if (edge) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int c8 = 0; c8 < NT; ++c8)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int at = key + 16 * m + g + 8 * (i >> 1);
              if (at >= min(limit[c8][i & 1], key1)) s[m][c8][i] = -INFINITY;
            }
        // weights of zero do not hide a NaN of V: values past the end become zero, a NaN that only some rows see is noted
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int at = key + 16 * m + 2 * t + (i & 1) + 8 * (i >> 1);
#pragma unroll
            for (int w = 0; w < VW; ++w) {
              if (at >= key1) vr[m][i][w] = 0u;
              const uint32_t nan = ((vr[m][i][w] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
              if (nan && p.n > 1) {
                for (int x = 0; x < 4; ++x)
                  if (nan >> (8 * x + 7) & 1u) {
                    atomicMin(&nan_key[v_dim(w) + x], at);
                    vr[m][i][w] &= ~(0xFFu << (8 * x));
                  }
              }
            }
          }
      }
      // ---- running reference and weights
      uint32_t pb[2][NT][2];
#pragma unroll
      for (int c8 = 0; c8 < NT; ++c8) {
        float mx[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) mx[i] = fmaxf(fmaxf(s[0][c8][i], s[0][c8][i + 2]), fmaxf(s[1][c8][i], s[1][c8][i + 2]));
#pragma unroll
        for (int x = 4; x < 32; x <<= 1)
#pragma unroll
          for (int i = 0; i < 2; ++i) mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], x));
        if (__any_sync(0xffffffffu, mx[0] > R[c8][0] || mx[1] > R[c8][1])) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float rn = fmaxf(R[c8][i], mx[i]), alpha = ex2_approx(R[c8][i] - rn);
            R[c8][i] = rn;
            l[c8][i] *= alpha;
#pragma unroll
            for (int w = 0; w < VW; ++w)
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                o[w][y][c8][i] *= alpha;
                o[w][y][c8][i + 2] *= alpha;
              }
          }
        }
        const float up[2] = {R[c8][0] - 15.f, R[c8][1] - 15.f};
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          float w4[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            w4[i] = ex2_approx(s[m][c8][i] - up[i & 1]);
            l[c8][i & 1] = fmaf(w4[i], cf[m], l[c8][i & 1]);
          }
          pb[m][c8][0] = transpose8x8(half2_bits(w4[0], w4[1]));
          pb[m][c8][1] = transpose8x8(half2_bits(w4[2], w4[3]));
        }
      }
      // ---- O^T += V^T P^T: a lane's words hold four channels of keys 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int w = 0; w < VW; ++w)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const uint32_t sel = y ? 0x7362u : 0x5140u;
            const uint32_t x0 = __byte_perm(vr[m][0][w], vr[m][1][w], sel), x1 = __byte_perm(vr[m][2][w], vr[m][3][w], sel);
            const uint32_t a[4] = {kv8_half2(x0, false), kv8_half2(x0, true), kv8_half2(x1, false), kv8_half2(x1, true)};
#pragma unroll
            for (int c8 = 0; c8 < NT; ++c8) mma_f16(o[w][y][c8], a, pb[m][c8][0], pb[m][c8][1]);
          }
      if (more) load_v(key + KA_STEP * KA_WARPS);
    }

    // ---- the warps' results meet in shared memory
#pragma unroll
    for (int c8 = 0; c8 < NT; ++c8) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float sum = l[c8][i];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        const int c = 8 * c8 + 2 * t + i;
        if (c < nrows) {
          if (g == 0) {
            sm_r[warp * p.rows + c] = R[c8][i];
            sm_l[warp * p.rows + c] = sum;
          }
#pragma unroll
          for (int w = 0; w < VW; ++w)
            *reinterpret_cast<float4*>(sm_o + (static_cast<size_t>(warp) * p.rows + c) * D + v_dim(w)) =
                make_float4(o[w][0][c8][i], o[w][0][c8][i + 2], o[w][1][c8][i], o[w][1][c8][i + 2]);
        }
      }
    }
    __syncthreads();
    const bool whole = t0 == 0 && t1 == nt;
    float* part = whole ? nullptr : p.part + (2ll * blockIdx.x + (t0 == 0 ? 1 : 0)) * p.rows * (D + 2);
    for (int x = threadIdx.x; x < nrows * (D / 4); x += 32 * KA_WARPS) {
      const int r = x / (D / 4), d = 4 * (x - r * (D / 4));
      float top = KA_NEG, sum = 0.f;
#pragma unroll
      for (int w = 0; w < KA_WARPS; ++w) top = fmaxf(top, sm_r[w * p.rows + r]);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < KA_WARPS; ++w) {
        const float f = ex2_approx(sm_r[w * p.rows + r] - top);
        const float4 y = *reinterpret_cast<const float4*>(sm_o + (static_cast<size_t>(w) * p.rows + r) * D + d);
        sum = fmaf(sm_l[w * p.rows + r], f, sum);
        acc.x = fmaf(y.x, f, acc.x); acc.y = fmaf(y.y, f, acc.y); acc.z = fmaf(y.z, f, acc.z); acc.w = fmaf(y.w, f, acc.w);
      }
      const int row = r0 + r, i = row / p.group, hq = h * p.group + row - i * p.group;
      if (p.n > 1) {
        const int sees = len - (p.n - 1) + i;
        if (nan_key[d] < sees) acc.x = NAN;
        if (nan_key[d + 1] < sees) acc.y = NAN;
        if (nan_key[d + 2] < sees) acc.z = NAN;
        if (nan_key[d + 3] < sees) acc.w = NAN;
      }
      if (whole) {
        const float f = sum == 0.f ? 0.f : 1.f / sum, e = pow2i(e_ref);
        *reinterpret_cast<uint2*>(p.out + ((static_cast<size_t>(b) * p.n + i) * p.Hkv * p.group + hq) * D + d) =
            make_uint2(pack_bf16x2(acc.x * f * e, acc.y * f * e), pack_bf16x2(acc.z * f * e, acc.w * f * e));
      } else {
        *reinterpret_cast<float2*>(part + r * (D + 2) + d) = make_float2(acc.x, acc.y);
        *reinterpret_cast<float2*>(part + r * (D + 2) + d + 2) = make_float2(acc.z, acc.w);
        if (d == 0) *reinterpret_cast<float2*>(part + r * (D + 2) + D) = make_float2(top, sum);
      }
    }
    __syncthreads();
    if (p.n > 1) {
      for (int d = threadIdx.x; d < D; d += 32 * KA_WARPS) nan_key[d] = INT_MAX;
      __syncthreads();
    }
  }
}

// Joins the partial results of ranges that several CTAs shared.  One warp per row of a range; grid (rows of a sequence / 4, B).
template <int D>
__global__ void __launch_bounds__(128)
kv8_join_kernel(const Kv8Attn p, int ctas) {
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.y, lane = threadIdx.x & 31, idx = blockIdx.x * 4 + (threadIdx.x >> 5);
  const Shares sh(p);
  const int nt = sh.tiles_of(p, b);
  if (nt == 1 || idx >= sh.per_unit * p.rows) return;
  const int unit = idx / p.rows, r = idx - unit * p.rows;
  const int h = unit / p.tiles_r, row = (unit - h * p.tiles_r) * p.rows + r;
  if (row >= p.n * p.group) return;
  const long long G = min(static_cast<long long>(ctas), sh.total), first = sh.base(p, b) + static_cast<long long>(unit) * nt;
  const int c0 = static_cast<int>(((first + 1) * G - 1) / sh.total), c1 = static_cast<int>(((first + nt) * G - 1) / sh.total);
  if (c0 == c1) return;                             // written by its CTA
  float acc[D / 32], top = KA_NEG, sum = 0.f;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) acc[i] = 0.f;
  for (int c = c0; c <= c1; ++c) {                  // the CTA that begins the range kept it in its second place
    const float* part = p.part + (2ll * c + (c == c0 ? 1 : 0)) * p.rows * (D + 2) + static_cast<long long>(r) * (D + 2);
    const float2 ml = *reinterpret_cast<const float2*>(part + D);
    const float tn = fmaxf(top, ml.x), f0 = ex2_approx(top - tn), f1 = ex2_approx(ml.x - tn);
    top = tn;
    sum = sum * f0 + ml.y * f1;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = acc[i] * f0 + part[lane + 32 * i] * f1;
  }
  const float f = sum == 0.f ? 0.f : 1.f / sum, e = pow2i(p.ve[b * p.eb + h * p.eh]);
  const int i = row / p.group, hq = h * p.group + row - i * p.group;
#pragma unroll
  for (int x = 0; x < D / 32; ++x)
    p.out[((static_cast<size_t>(b) * p.n + i) * p.Hkv * p.group + hq) * D + lane + 32 * x] = f2bf(acc[x] * f * e);
}

template <int D, int NT>
static int kv8_smem(int rows) {
  return 4 * KA_WARPS * rows * (D + 2) + (NT > 1 ? NT * (D / 16) * 32 * 8 + 8 * NT * 4 : 0);
}

template <int D, int NT>
static int kv8_slots(int rows) {                    // CTAs that one SM holds
  auto kern = kv8_attention_kernel<D, NT>;
  int dev = 0, per = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  static int known[64][33] = {};
  if (!known[dev][rows]) {
    const int smem = kv8_smem<D, NT>(rows);
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 4 * KA_WARPS * 8 * NT * (D + 2) + NT * (D / 16) * 32 * 8 + 8 * NT * 4) != cudaSuccess ||
        cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kern, 32 * KA_WARPS, smem) != cudaSuccess || per < 1)
      return 0;
    known[dev][rows] = per;
  }
  return known[dev][rows];
}

template <int D>
static int kv8_slots_d(int nt, int rows) {
  switch (nt) {
    case 1: return kv8_slots<D, 1>(rows);
    case 2: return kv8_slots<D, 2>(rows);
    case 3: return kv8_slots<D, 3>(rows);
    case 4: return kv8_slots<D, 4>(rows);
    default: return 0;
  }
}
static int kv8_slots_any(int D, int nt, int rows) {
  switch (D) {
    case 32: return kv8_slots_d<32>(nt, rows);
    case 64: return kv8_slots_d<64>(nt, rows);
    case 96: return kv8_slots_d<96>(nt, rows);
    case 128: return kv8_slots_d<128>(nt, rows);
    default: return 0;
  }
}

template <int D>
static void kv8_run(const Kv8Attn& p, int nt, int ctas, cudaStream_t st) {
  const dim3 block(32 * KA_WARPS);
  if (nt == 1) launch_k(kv8_attention_kernel<D, 1>, dim3(ctas), block, kv8_smem<D, 1>(p.rows), st, p);
  else if (nt == 2) launch_k(kv8_attention_kernel<D, 2>, dim3(ctas), block, kv8_smem<D, 2>(p.rows), st, p);
  else if (nt == 3) launch_k(kv8_attention_kernel<D, 3>, dim3(ctas), block, kv8_smem<D, 3>(p.rows), st, p);
  else launch_k(kv8_attention_kernel<D, 4>, dim3(ctas), block, kv8_smem<D, 4>(p.rows), st, p);
  if (p.part) launch_k(kv8_join_kernel<D>, dim3((p.Hkv * p.tiles_r * p.rows + 3) / 4, p.B), dim3(128), 0, st, p, ctas);
}

}  // namespace b200

using namespace b200;

// How a call is cut.  plan: [0] rows per row tile, [1] row tiles, [2] keys per tile, [3] CTAs, [4] floats of scratch (0: none).
B200_API int b200_kv8_attention_plan(int B, int Hkv, int D, int rows, int most, int* plan) {
  if (B <= 0 || B > 65535 || Hkv <= 0 || rows <= 0 || most <= 0) return -1;
  const int tiles_r = (rows + 31) / 32, per = (rows + tiles_r - 1) / tiles_r;
  const int slots = kv8_slots_any(D, (per + 7) / 8, per);
  if (!slots) return -2;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return -3;
  const long long ranges = static_cast<long long>(B) * Hkv * tiles_r;
  const int tile = most <= 512 ? 512 : KA_WARPS * KA_STEP;
  const long long tiles = ranges * ((most + tile - 1) / tile);
  if (tiles / B > (1ll << 31) - 1 || ranges > (1ll << 31) - 1) return -4;
  const bool whole = tile >= most;
  const long long ctas = whole ? tiles : (tiles < static_cast<long long>(sms) * slots ? tiles : static_cast<long long>(sms) * slots);
  plan[0] = per;
  plan[1] = tiles_r;
  plan[2] = tile;
  plan[3] = static_cast<int>(ctas);
  plan[4] = whole ? 0 : static_cast<int>(ctas * 2 * per * (D + 2));
  return 0;
}

// p as in Kv8Attn (rows, tiles_r, tile as planned); ctas from the plan.
B200_API int b200_kv8_attention(const Kv8Attn* a, int ctas, void* stream) {
  const Kv8Attn& p = *a;
  if (p.B <= 0 || p.B > 65535 || p.Hkv <= 0 || p.n <= 0 || p.group <= 0 || p.rows <= 0 || p.rows > 32 || p.tiles_r <= 0 || ctas <= 0 ||
      p.log2_block < 4 || p.log2_block > 7 || p.most <= 0 || p.most > p.cap || p.tile % (KA_WARPS * KA_STEP) || (!p.part && p.tile < p.most))
    return -1;
  if (static_cast<long long>(p.rows) * p.tiles_r < static_cast<long long>(p.n) * p.group) return -1;
  if ((reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v) | p.sb | p.sh) & 15) return -2;
  if (((reinterpret_cast<uintptr_t>(p.q) | reinterpret_cast<uintptr_t>(p.out)) & 15) || ((p.q_sb | p.q_sn | p.q_sh) & 7)) return -2;
  if (!kv8_slots_any(p.D, (p.rows + 7) / 8, p.rows)) return -3;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int nt = (p.rows + 7) / 8;
  switch (p.D) {
    case 32: kv8_run<32>(p, nt, ctas, st); break;
    case 64: kv8_run<64>(p, nt, ctas, st); break;
    case 96: kv8_run<96>(p, nt, ctas, st); break;
    case 128: kv8_run<128>(p, nt, ctas, st); break;
    default: return -1;
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -10;
}
