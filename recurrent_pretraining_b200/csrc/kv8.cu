// Writing and reading the 8-bit key / value cache (kv8.cuh):
//   * kv8_append       : n tokens per sequence, any start, one CTA per (sequence, head, touched block, keys or values)
//   * kv8_rope_append  : the one new token of a decode step from its packed projection: bias, rotation, q out, k and v encoded
//   * kv8_decode       : codes back to bf16 rows [B, L, Hkv, D] (exact), as the prompt attention reads them
//   * kv8_tiles        : tile table of the prompt attention, from the lengths on the device
//   * kv8_nan          : NaNs of V among a prompt's own tokens, put into the rows that see them
//
// A block that is begun takes the exponent of its new tokens, so what lay in the cache before does not matter and freed rows need
// no clearing.  A block that goes on keeps the larger of both exponents; when the new tokens' is larger, what it holds in front of
// them is encoded again by the CTA (or lane group) that writes them.  Writing the same tokens to the same place again
// changes nothing: exponents only grow.  Nothing behind the new tokens is touched.
//
// Appending is bound by memory: 4 x 1024 tokens of 55 heads of 96 take 22.0 us, 5.9 TB/s of reads and writes mixed (28.1 with the magnitudes
// compared as fp32 numbers: there were more instructions than the memory left time for).  A step's tokens (64 sequences, 48
// heads of 128) take 2.6 us, about an empty launch.
#include <algorithm>

#include "kv8.cuh"

namespace b200 {

struct Kv8Cache {
  uint8_t *k, *v;                    // codes
  int8_t *ke, *ve;                   // exponents
  long long sb, sh, eb, eh;          // batch and head pitch of codes and exponents (elements)
  int B, Hkv, cap, D, log2_block;
};

// Threads for a block of so many values, 16 to 96 values each.  4 x 1024 tokens of 5280 channels (the one shape that the borders were measured at; a
// call of few tokens is bound by its launch), 20 us of copying: 20.1 to 22.3 us with every block and dim but 16 x 32 (25.1).  2048 values take 25.5 with 128 threads, 23.7 with 64, 21.8 with a warp; 16384 take 26.3 with 128 threads, 20.7 with 256.
__host__ __device__ constexpr int kv8_group(int values) { return values <= 2048 ? 32 : values <= 12288 ? 128 : 256; }
__host__ __device__ constexpr int kv8_threads(int G) { return G > 32 ? G : 128; }

// grid (2 x most touched blocks / (threads / G), Hkv, B), kv8_threads(G) threads, G of them (a warp or the CTA) per block of BLK tokens.  The block's new tokens
// stay in registers (NV vectors of eight values per thread) between the maximum and the encoding: one pass over the input.  D and BLK
// are known to the compiler: a division per vector would take longer than the vector.
template <int D, int BLK, int G>
__global__ void __launch_bounds__(kv8_threads(G))
kv8_append_kernel(const Kv8Cache c, const __nv_bfloat16* __restrict__ k, const __nv_bfloat16* __restrict__ v, long long k_sb,
                  long long k_sn, long long k_sh, long long v_sb, long long v_sn, long long v_sh, const int* __restrict__ start_,
                  const int* __restrict__ counts, int n, int* err) {
  pdl_trigger();
  pdl_wait();
  const int unit = blockIdx.x * (kv8_threads(G) / G) + threadIdx.x / G, which = unit & 1, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x % G;
  const int start = start_[b], cnt = counts ? counts[b] : n;
  if (start < 0 || cnt < 0 || cnt > n || start > c.cap - cnt) {     // the sequence does not fit: nothing of it is written
    if (tid == 0 && err) atomicCAS(err, 0, ERR_BAD_INDEX);
    return;
  }
  const int block = start / BLK + (unit >> 1), p0 = block * BLK;
  const int lo = max(start, p0), hi = min(start + cnt, p0 + BLK);
  if (lo >= hi) return;
  const long long sn = which ? v_sn : k_sn;
  const __nv_bfloat16* src = (which ? v + b * v_sb + h * v_sh : k + b * k_sb + h * k_sh) + (lo - start) * sn;
  uint8_t* dst = (which ? c.v : c.k) + b * c.sb + h * c.sh + static_cast<long long>(p0) * D;
  int8_t* ep = (which ? c.ve : c.ke) + b * c.eb + h * c.eh + block;
  constexpr int vpr = D / 8, NV = (BLK * vpr + G - 1) / G;
  const int nvec = (hi - lo) * vpr;
  uint4 x[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int idx = tid + G * i;
    x[i] = make_uint4(0u, 0u, 0u, 0u);
    if (idx < nvec) x[i] = __ldg(reinterpret_cast<const uint4*>(src + (idx / vpr) * sn) + idx % vpr);
  }
  const bool fresh = lo == p0;
  const int old = fresh ? KV8_EMIN : *ep;
  // magnitudes are compared in pairs of bf16; where there is an infinity or NaN, which do not count, one by one
  __nv_bfloat162 top = __float2bfloat162_rn(0.f);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) top = __hmax2_nan(top, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[j])));
  }
  float amax = __bfloat162float(__hmax_nan(__low2bfloat16(top), __high2bfloat16(top)));
  if (!(amax < INFINITY)) {
    amax = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const uint32_t w[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = unpack_bf16x2(w[j]);
        amax = fmaxf(amax, fmaxf(kv8_mag(f.x), kv8_mag(f.y)));
      }
    }
  }
  amax = warp_max(amax);                                            // every thread has read the old exponent, too
  if constexpr (G > 32) {
    __shared__ float red[G / 32];
    if ((tid & 31) == 0) red[tid >> 5] = amax;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < G / 32; ++i) amax = fmaxf(amax, red[i]);
  }
  const int e = max(kv8_exponent(amax), old);
  const float inv = pow2i(-e);
  if (tid == 0) *ep = static_cast<int8_t>(e);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int idx = tid + G * i;
    if (idx < nvec) {
      const float2 f0 = unpack_bf16x2(x[i].x), f1 = unpack_bf16x2(x[i].y), f2 = unpack_bf16x2(x[i].z), f3 = unpack_bf16x2(x[i].w);
      *reinterpret_cast<uint2*>(dst + static_cast<size_t>(lo - p0) * D + 8 * static_cast<size_t>(idx)) =
          make_uint2(kv8_encode4(f0.x, f0.y, f1.x, f1.y, inv), kv8_encode4(f2.x, f2.y, f3.x, f3.y, inv));
    }
  }
  if (!fresh && e > old) {
    const float f = pow2i(old - e);
    for (int idx = tid; idx < (lo - p0) * vpr; idx += G) {
      uint2* w = reinterpret_cast<uint2*>(dst) + idx;
      *w = make_uint2(kv8_recode4(w->x, f), kv8_recode4(w->y, f));
    }
  }
}

// One group of 16 lanes per (sequence, head of q, k or v), eight channels per lane.  F32_IN: the projection is an fp32 accumulator,
// handed back zeroed when `clear` is set.  Values reach the codes from fp32 directly (one rounding); q is rounded once, to bf16.
template <bool F32_IN>
__global__ void __launch_bounds__(256)
kv8_rope_append_kernel(const Kv8Cache c, void* __restrict__ qkv, long long ld, const float* __restrict__ bias,
                       const float* __restrict__ cosT, const float* __restrict__ sinT, const int* __restrict__ pos,
                       __nv_bfloat16* __restrict__ q_out, int H, int clear, int* err) {
  pdl_trigger();
  const int heads = H + 2 * c.Hkv;
  const int unit = blockIdx.x * 16 + (threadIdx.x >> 4), j = threadIdx.x & 15;
  const bool live = unit < c.B * heads && 8 * j < c.D;
  const int b = live ? unit / heads : 0, hh = live ? unit - b * heads : 0;
  const bool rotated = hh < H + c.Hkv;
  pdl_wait();
  float add[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) add[i] = live && rotated && bias ? bias[hh * c.D + 8 * j + i] : 0.f;
  const int p = live ? pos[b] : 0;
  const bool ok = live && p >= 0 && p < c.cap;
  if (live && !ok && err) atomicCAS(err, 0, ERR_BAD_INDEX);
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = 0.f;
  if (live) {
    if constexpr (F32_IN) {
      float4* src = reinterpret_cast<float4*>(static_cast<float*>(qkv) + b * ld + hh * c.D + 8 * j);
      const float4 a = src[0], d = src[1];
      if (clear) src[0] = src[1] = make_float4(0.f, 0.f, 0.f, 0.f);
      x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = d.x; x[5] = d.y; x[6] = d.z; x[7] = d.w;
    } else {
      const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(qkv) + b * ld + hh * c.D + 8 * j);
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack_bf16x2(w[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  }
  if (ok && rotated) {
    const float4 cs = *reinterpret_cast<const float4*>(cosT + static_cast<size_t>(p) * (c.D >> 1) + 4 * j);
    const float4 sn = *reinterpret_cast<const float4*>(sinT + static_cast<size_t>(p) * (c.D >> 1) + 4 * j);
    const float cw[4] = {cs.x, cs.y, cs.z, cs.w}, sw[4] = {sn.x, sn.y, sn.z, sn.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float u = x[2 * i] + add[2 * i], w = x[2 * i + 1] + add[2 * i + 1];
      x[2 * i] = u * cw[i] - w * sw[i];
      x[2 * i + 1] = w * cw[i] + u * sw[i];
    }
  }
  float amax = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) amax = fmaxf(amax, kv8_mag(x[i]));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  const int which = hh >= H + c.Hkv, h = hh - H - which * c.Hkv;    // of a key or value head
  const int block = p >> c.log2_block, p0 = block << c.log2_block;
  int8_t* ep = nullptr;
  int old = KV8_EMIN;
  if (ok && hh >= H) {
    ep = (which ? c.ve : c.ke) + b * c.eb + h * c.eh + block;
    if (p > p0) old = *ep;
  }
  __syncwarp();                                                     // the group has read the exponent
  if (!ok) return;
  if (hh < H) {
    *reinterpret_cast<uint4*>(q_out + (static_cast<size_t>(b) * H + hh) * c.D + 8 * j) =
        make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
    return;
  }
  const int e = max(kv8_exponent(amax), old);
  const float inv = pow2i(-e);
  uint8_t* dst = (which ? c.v : c.k) + b * c.sb + h * c.sh + static_cast<long long>(p0) * c.D + 8 * j;
  *reinterpret_cast<uint2*>(dst + (p - p0) * c.D) = make_uint2(kv8_encode4(x[0], x[1], x[2], x[3], inv), kv8_encode4(x[4], x[5], x[6], x[7], inv));
  if (j == 0) *ep = static_cast<int8_t>(e);
  if (p > p0 && e > old) {
    const float f = pow2i(old - e);
    for (int t = 0; t < p - p0; ++t) {
      uint2* w = reinterpret_cast<uint2*>(dst + t * c.D);
      *w = make_uint2(kv8_recode4(w->x, f), kv8_recode4(w->y, f));
    }
  }
}

// out rows [B * L, ld], head h at column h * D: keys (blockIdx.y 0) and values (1) of positions below L.  With `lens`, positions from the
// length to the next multiple of 128 become zero (an attention tile that ends there reads them) and later ones are left out.  `nan_first`: a weight
// of zero does not hide a NaN of V from the queries in front of it, so NaNs among the newest n positions become zero and are noted there.
__global__ void __launch_bounds__(256)
kv8_decode_kernel(const Kv8Cache c, const int* __restrict__ lens, __nv_bfloat16* __restrict__ k_out, __nv_bfloat16* __restrict__ v_out,
                  int L, int most, int ld, int* __restrict__ nan_first, int n) {
  pdl_trigger();
  pdl_wait();
  const int vpr = c.D >> 3, per_row = c.Hkv * vpr, b = blockIdx.z;
  const long long idx = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const int t0 = 4 * static_cast<int>(idx / per_row), col = static_cast<int>(idx - static_cast<long long>(t0 / 4) * per_row);   // tokens t0 .. t0 + 3, eight channels
  const int len = lens ? min(max(lens[b], 0), most) : L;
  const int end = min(L, (len + 127) & ~127);
  if (t0 >= end) return;
  const int h = col / vpr, d = (col - h * vpr) * 8;
  const uint8_t* src = (blockIdx.y ? c.v : c.k) + b * c.sb + h * c.sh + static_cast<long long>(t0) * c.D + d;
  __nv_bfloat16* dst = (blockIdx.y ? v_out : k_out) + (static_cast<long long>(b) * L + t0) * ld + h * c.D + d;
  uint2 w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = t0 + i < len ? __ldg(reinterpret_cast<const uint2*>(src + i * c.D)) : make_uint2(0u, 0u);
  const float f = t0 < len ? pow2i((blockIdx.y ? c.ve : c.ke)[b * c.eb + h * c.eh + (t0 >> c.log2_block)]) : 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (t0 + i >= end) break;
    if (nan_first && blockIdx.y && t0 + i >= len - n) {
      const unsigned long long all = w[i].x | (static_cast<unsigned long long>(w[i].y) << 32);
      unsigned long long keep = ~0ull;
      if (((all & 0x7F7F7F7F7F7F7F7Full) + 0x0101010101010101ull) & 0x8080808080808080ull)
        for (int x = 0; x < 8; ++x)
          if ((all >> (8 * x) & 0x7F) == 0x7F) {
            keep &= ~(0xFFull << (8 * x));
            atomicMin(nan_first + (static_cast<long long>(b) * c.Hkv + h) * c.D + d + x, t0 + i);
          }
      w[i].x &= static_cast<uint32_t>(keep);
      w[i].y &= static_cast<uint32_t>(keep >> 32);
    }
    const float2 a0 = kv8_float2(w[i].x, false), a1 = kv8_float2(w[i].x, true), a2 = kv8_float2(w[i].y, false), a3 = kv8_float2(w[i].y, true);
    *reinterpret_cast<uint4*>(dst + static_cast<long long>(i) * ld) =
        make_uint4(pack_bf16x2(a0.x * f, a0.y * f), pack_bf16x2(a1.x * f, a1.y * f), pack_bf16x2(a2.x * f, a2.y * f), pack_bf16x2(a3.x * f, a3.y * f));
  }
}

// One CTA per (sequence, 256-query tile): {first query token, queries, stream index of the first query, first key of the sequence}, the tiles
// that see most keys first.  Queries in front of the sequence's first key have nothing to see: they are not in a tile and their outputs
// become zero here, and the table of NaNs (`noted` entries per sequence) is cleared.
__global__ void __launch_bounds__(256)
kv8_tiles_kernel(const int* __restrict__ lens, int4* __restrict__ tiles, __nv_bfloat16* __restrict__ out, int n, int most, int L, int per_seq, long long row,
                 int* __restrict__ nan_first, int noted) {
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.x, i = blockIdx.y, B = gridDim.x;
  const int len = min(max(lens[b], 0), most), skip = max(0, n - len);  // queries that see nothing
  const int q = skip + 256 * i, rows = max(0, min(256, n - q));
  if (threadIdx.x == 0)
    tiles[(per_seq - 1 - i) * B + b] = make_int4(b * n + (rows ? q : 0), rows, b * L + (rows ? len - n + q : 0), b * L);
  uint4* o = reinterpret_cast<uint4*>(out + static_cast<long long>(b) * n * row);
  const long long last = skip * row / 8;
  for (long long x = static_cast<long long>(i) * 256 + threadIdx.x; x < last; x += 256ll * per_seq) o[x] = make_uint4(0u, 0u, 0u, 0u);
  if (i == 0)
    for (int x = threadIdx.x; x < noted; x += 256) nan_first[static_cast<long long>(b) * noted + x] = INT_MAX;
}

// A thread per channel of a key head: the outputs [B, n, .., D] (pitch `row` per token) of the queries that see its first noted NaN.
__global__ void __launch_bounds__(128)
kv8_nan_kernel(const int* __restrict__ nan_first, const int* __restrict__ lens, __nv_bfloat16* __restrict__ out, int n, int group, int Hkv, int D, int most,
               long long row) {
  pdl_trigger();
  pdl_wait();
  const int b = blockIdx.y, h = blockIdx.x, d = threadIdx.x;
  if (d >= D) return;
  const int first = nan_first[(static_cast<long long>(b) * Hkv + h) * D + d];
  if (first == INT_MAX) return;
  const int len = min(max(lens[b], 0), most);
  for (int i = max(0, first - (len - n)); i < n; ++i)
    for (int x = 0; x < group; ++x) out[(static_cast<long long>(b) * n + i) * row + (h * group + x) * D + d] = __float2bfloat16(NAN);
}

}  // namespace b200

using namespace b200;

static bool kv8_cache_ok(const Kv8Cache* c) {
  return c->k && c->v && c->ke && c->ve && c->B > 0 && c->B <= 65535 && c->Hkv > 0 && c->Hkv <= 65535 && c->D >= 32 && c->D <= 128 &&
         c->D % 32 == 0 && c->log2_block >= 4 && c->log2_block <= 7 && c->cap > 0 && c->cap % (1 << c->log2_block) == 0 &&
         !((reinterpret_cast<uintptr_t>(c->k) | reinterpret_cast<uintptr_t>(c->v)) & 15) && !((c->sb | c->sh) & 15);
}

// k, v: [B, n, Hkv, D] bf16 with pitches in elements (three each, multiples of eight); start, counts (null: n each): [B].
B200_API int b200_kv8_append(const Kv8Cache* c, const void* k, const void* v, const long long* pitch, const int* start, const int* counts, int n,
                             int* err, void* stream) {
  if (!kv8_cache_ok(c) || n <= 0) return -1;
  for (int i = 0; i < 6; ++i)
    if (pitch[i] & 7) return -2;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) return -2;
  const int blk = 1 << c->log2_block;
  const long long touched = (static_cast<long long>(n) + blk - 2) / blk + 1;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const __nv_bfloat16 *kb = static_cast<const __nv_bfloat16*>(k), *vb = static_cast<const __nv_bfloat16*>(v);
#define RUN(D, BLK) \
  case D * 1000 + BLK: { \
    constexpr int G = kv8_group(BLK * D), per = kv8_threads(G) / G; \
    launch_k(kv8_append_kernel<D, BLK, G>, dim3(static_cast<unsigned>((2 * touched + per - 1) / per), c->Hkv, c->B), dim3(kv8_threads(G)), 0, st, *c, kb, vb, \
             pitch[0], pitch[1], pitch[2], pitch[3], pitch[4], pitch[5], start, counts, n, err); \
    break; \
  }
#define RUN_D(D) RUN(D, 16) RUN(D, 32) RUN(D, 64) RUN(D, 128)
  switch (c->D * 1000 + blk) {
    RUN_D(32) RUN_D(64) RUN_D(96) RUN_D(128)
    default: return -1;
  }
#undef RUN_D
#undef RUN
  return cudaGetLastError() == cudaSuccess ? 0 : -10;
}

// qkv: [B, ld] = [q heads | k heads | v heads], bf16 or fp32; bias: fp32 [(H + Hkv) D] or null; cos / sin: fp32 [>= cap, D / 2]; pos: [B].
B200_API int b200_kv8_rope_append(const Kv8Cache* c, void* qkv, long long ld, int is_f32, int clear, const float* bias, const float* cosT,
                                  const float* sinT, const int* pos, void* q_out, int H, int* err, void* stream) {
  if (!kv8_cache_ok(c) || H <= 0) return -1;
  if ((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(cosT) | reinterpret_cast<uintptr_t>(sinT)) & 15) return -2;
  if (ld & (is_f32 ? 3 : 7)) return -2;
  const long long units = static_cast<long long>(c->B) * (H + 2 * c->Hkv);
  if (units > (1ll << 31) - 16) return -3;
  const dim3 grid(static_cast<unsigned>((units + 15) / 16));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  __nv_bfloat16* qo = static_cast<__nv_bfloat16*>(q_out);
  if (is_f32) launch_k(kv8_rope_append_kernel<true>, grid, dim3(256), 0, st, *c, qkv, ld, bias, cosT, sinT, pos, qo, H, clear, err);
  else launch_k(kv8_rope_append_kernel<false>, grid, dim3(256), 0, st, *c, qkv, ld, bias, cosT, sinT, pos, qo, H, clear, err);
  return cudaGetLastError() == cudaSuccess ? 0 : -10;
}

// k_out, v_out: bf16 [B, L, Hkv, D] contiguous, lens, nan_first (int32 [B, Hkv, D], cleared; or null), n: see kv8_decode_kernel (no length counts for
// more than `most`).
B200_API int b200_kv8_decode(const Kv8Cache* c, const int* lens, void* k_out, void* v_out, int L, int most, int* nan_first, int n, void* stream) {
  if (!kv8_cache_ok(c) || L <= 0 || most > L || most > c->cap || (!lens && L > c->cap)) return -1;
  if ((reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) & 15) return -2;
  const long long vecs = static_cast<long long>((L + 3) / 4) * c->Hkv * (c->D / 8);
  if (vecs > (1ll << 38)) return -3;
  launch_k(kv8_decode_kernel, dim3(static_cast<unsigned>((vecs + 255) / 256), 2, c->B), dim3(256), 0, reinterpret_cast<cudaStream_t>(stream), *c, lens,
           static_cast<__nv_bfloat16*>(k_out), static_cast<__nv_bfloat16*>(v_out), L, most, c->Hkv * c->D, lens ? nan_first : nullptr, n);
  return cudaGetLastError() == cudaSuccess ? 0 : -10;
}

// ---- a prompt's attention: the codes become bf16 rows, which the tensor-core attention of latent_attention.cu reads
B200_API int b200_attention_parts(int n_tiles, int H, int keys);
B200_API int b200_capped_attention(const void* q, const void* k, const void* v, void* out, const int* tiles, const float* sink, int n_tiles, int T,
                                   int K, int H, int G, int dim, int vdim, int ld_q, int ld_kv, int ld_out, int window, int keep,
                                   float scale, float softcap, float bound, void* stream, int* err);
B200_API int b200_parted_attention(const void* q, const void* k, const void* v, void* out, const int* tiles, void* part_o, void* part_ml, int parts,
                                   int n_tiles, int T, int K, int H, int G, int dim, int vdim, int ld_q, int ld_kv, int ld_out, float scale,
                                   void* stream, int* err);

// Sequences and key heads are answered group by group through the same scratch memory, so that its size does not follow batch and capacity.
struct Kv8Prompt {
  int L, per_seq;                                 // key rows and query tiles per sequence
  int seqs, heads;                                // of a group: sequences, key heads
  size_t bytes;                                   // of scratch memory
};
struct Kv8Places {
  int parts;                                      // CTAs per tile
  size_t v, tiles, nans, refs, sums, bytes;       // places in the scratch memory; keys are first
};
static Kv8Places kv8_prompt_places(const Kv8Prompt& x, int seqs, int heads, int group, int D, int most) {
  Kv8Places at = {};
  const long long W = static_cast<long long>(heads) * D, n_tiles = static_cast<long long>(seqs) * x.per_seq, H = static_cast<long long>(heads) * group;
  at.parts = b200_attention_parts(static_cast<int>(n_tiles), static_cast<int>(H), most);
  auto place = [&](size_t bytes) { const size_t p = at.bytes; at.bytes += (bytes + 255) & ~size_t(255); return p; };
  const size_t rows = static_cast<size_t>(seqs) * x.L * W * 2, cells = at.parts > 1 ? static_cast<size_t>(n_tiles) * H * at.parts * 256 : 0;
  place(rows);
  at.v = place(rows);
  at.tiles = place(n_tiles * 16);
  at.nans = place(static_cast<size_t>(seqs) * W * 4);
  at.refs = place(cells * 8);
  at.sums = place(cells * D * 4);
  return at;
}
// Groups that need at most `limit` bytes, or one key head of one sequence.  Whole sequences, as long as there is room: their tiles fill the machine sooner.
static bool kv8_prompt_plan(Kv8Prompt* x, int B, int Hkv, int H, int D, int n, int most, long long limit) {
  if (most > INT_MAX - 127 || n > INT_MAX - 255 || static_cast<long long>(H) * D > INT_MAX) return false;
  x->L = (most + 127) & ~127;
  x->per_seq = (n + 255) / 256;
  const int fit = std::min((65535 / 4) / x->per_seq, INT_MAX / std::max(x->L, n));       // tiles in a grid, rows in 31 bits
  if (fit < 1) return false;
  x->seqs = std::min(B, fit);
  x->heads = Hkv;
  auto need = [&] {                               // of the full groups and of those that are left over
    size_t most_bytes = 0;
    for (int seqs : {x->seqs, B % x->seqs})
      for (int heads : {x->heads, Hkv % x->heads})
        if (seqs && heads) most_bytes = std::max(most_bytes, kv8_prompt_places(*x, seqs, heads, H / Hkv, D, most).bytes);
    return most_bytes;
  };
  while ((x->bytes = need()) > static_cast<size_t>(std::max(limit, 0ll)) && (x->seqs > 1 || x->heads > 1)) {
    if (x->seqs > 1) x->seqs = (x->seqs + 1) / 2;
    else x->heads = (x->heads + 1) / 2;
  }
  return true;
}

// Bytes of scratch memory, at most `limit` where a key head of a sequence does not take more; 0: too many tokens for the attention of tiles.
B200_API long long b200_kv8_prompt_scratch(int B, int Hkv, int H, int D, int n, int most, long long limit) {
  Kv8Prompt x;
  if (B <= 0 || Hkv <= 0 || H <= 0 || H % Hkv || D <= 0 || n <= 0 || most <= 0 || !kv8_prompt_plan(&x, B, Hkv, H, D, n, most, limit)) return 0;
  return static_cast<long long>(x.bytes);
}

// q, out: bf16 [B, n, H, D] contiguous; no length counts for more than `most`; scratch as above.
B200_API int b200_kv8_prompt(const Kv8Cache* c, const void* q, const int* lens, void* out, void* scratch, int H, int n, int most, float scale,
                             long long limit, int* err, void* stream) {
  Kv8Prompt x;
  if (!kv8_cache_ok(c) || H <= 0 || H % c->Hkv || n <= 0 || most <= 0 || most > c->cap || !scratch ||
      !kv8_prompt_plan(&x, c->B, c->Hkv, H, c->D, n, most, limit))
    return -1;
  if (reinterpret_cast<uintptr_t>(scratch) & 255) return -2;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const int D = c->D, group = H / c->Hkv;
  const long long row = static_cast<long long>(H) * D;
  char* mem = static_cast<char*>(scratch);
  for (int b0 = 0; b0 < c->B; b0 += x.seqs)
    for (int h0 = 0; h0 < c->Hkv; h0 += x.heads) {
      Kv8Cache part = *c;                         // the group's sequences and key heads
      part.B = std::min(x.seqs, c->B - b0);
      part.Hkv = std::min(x.heads, c->Hkv - h0);
      part.k += b0 * c->sb + h0 * c->sh;
      part.v += b0 * c->sb + h0 * c->sh;
      part.ke += b0 * c->eb + h0 * c->eh;
      part.ve += b0 * c->eb + h0 * c->eh;
      const Kv8Places at = kv8_prompt_places(x, part.B, part.Hkv, group, D, most);
      const int W = part.Hkv * D, n_tiles = part.B * x.per_seq, heads = part.Hkv * group;
      int *tiles = reinterpret_cast<int*>(mem + at.tiles), *nans = reinterpret_cast<int*>(mem + at.nans);
      const __nv_bfloat16* qg = static_cast<const __nv_bfloat16*>(q) + static_cast<long long>(b0) * n * row + static_cast<long long>(h0) * group * D;
      __nv_bfloat16 *rows = static_cast<__nv_bfloat16*>(out) + static_cast<long long>(b0) * n * row, *og = rows + static_cast<long long>(h0) * group * D;
      // all heads' outputs of queries without keys become zero with the first group of heads
      launch_k(kv8_tiles_kernel, dim3(part.B, x.per_seq), dim3(256), 0, st, lens + b0, reinterpret_cast<int4*>(tiles), rows, n, most, x.L, x.per_seq,
               h0 ? 0ll : row, nans, W);
      int rc = b200_kv8_decode(&part, lens + b0, mem, mem + at.v, x.L, most, nans, n, stream);
      if (rc) return rc;
      if (at.parts > 1)
        rc = b200_parted_attention(qg, mem, mem + at.v, og, tiles, mem + at.sums, mem + at.refs, at.parts, n_tiles, part.B * n, part.B * x.L, heads, part.Hkv, D,
                                   D, H * D, W, H * D, scale, stream, err);
      else
        rc = b200_capped_attention(qg, mem, mem + at.v, og, tiles, nullptr, n_tiles, part.B * n, part.B * x.L, heads, part.Hkv, D, D, H * D, W, H * D, 1 << 30, 0,
                                   scale, 0.f, 0.f, stream, err);
      if (rc) return rc - 100;
      launch_k(kv8_nan_kernel, dim3(part.Hkv, part.B), dim3(128), 0, st, nans, lens + b0, og, n, group, part.Hkv, D, most, row);
    }
  return cudaGetLastError() == cudaSuccess ? 0 : -10;
}
