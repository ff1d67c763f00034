// A 4-bit paged KV cache written as the projection's rows are formed, and the read-back of any cache.
#include "common.h"
#include "kv4.h"
#include "kv4_entry.h"
#include "kvrow.h"

namespace dsk {

// ----------------------------------------------------------------------------- append
// q, k: x * rsqrt(mean(x^2) + eps) * w, rotated by pos * inv_freq; k and v to 4-bit codes (kv4.h). A row is not
// rounded between its projection's sum and its code or its bf16 query: to bf16, that would move about one code
// in a hundred. Keys are formed in 64 bits, and so are the sums of slices: in 32, a few of the codes of a
// 2048-token prompt are not the nearest (1.4 us more for 40 heads of 128 with 8 of V).
//
// What bounds it: few rows, the chain of loads (lengths, row, angles: 6.6 us for one token in a graph, of which
// about 4 are two launches); many, the bytes: 44 MB for that prompt, 14.6 us, 3.0 TB/s.
//
// Queries and keys: one workgroup per token row and chunk of heads; the row's HD / 2 sines and cosines are found
// once, one per thread, for all heads of the chunk; then 8 dims per lane, HD / 8 lanes per head. V, in the same
// launch: one workgroup per 4 positions.

// sin and cos of p f, p an integer and f a float32 (a float32 angle would be off by up to 2^-25 of itself: 0.004
// rad at position 131072). The product is exact in 64 bits for p below 2^29. Reduction by a multiple k of pi/2 =
// P1 + P2 (P1 its nearest double, the product inside the fma): off by 2^-53 of the remainder and k 2^-107. Then
// the Taylor polynomials on [-pi/4, pi/4], whose next terms are 2e-17 (sin, r^17 / 17!) and 5e-17 (cos).
__device__ __forceinline__ double2 rope_angle(double p, float f) {
  const double a = p * (double)f, k = rint(a * 0.63661977236758134308);
  const double r = fma(-k, 6.12323399573676588613e-17, fma(-k, 1.57079632679489661923, a)), z = r * r;
  double s = -7.6471637318198164759e-13, c = -1.1470745597729724714e-11;
  s = fma(s, z, 1.6059043836821614599e-10);
  s = fma(s, z, -2.5052108385441718775e-8);
  s = fma(s, z, 2.7557319223985890653e-6);
  s = fma(s, z, -1.9841269841269841270e-4);
  s = fma(s, z, 8.3333333333333333333e-3);
  s = fma(s, z, -1.6666666666666666667e-1);
  s = fma(s * z, r, r);
  c = fma(4.7794773323873852974e-14, z, c);
  c = fma(c, z, 2.0876756987868098979e-9);
  c = fma(c, z, -2.7557319223985890653e-7);
  c = fma(c, z, 2.4801587301587301587e-5);
  c = fma(c, z, -1.3888888888888888889e-3);
  c = fma(c, z, 4.1666666666666666667e-2);
  c = fma(c, z, -0.5);
  c = fma(c, z, 1.0);
  const int q = (int)((long long)k & 3);
  const double u = q & 1 ? c : s, v = q & 1 ? s : c;
  return double2{q == 1 || q == 2 ? -v : v, q & 2 ? -u : u};  // cos, sin
}

struct Kv4Append {
  const void* qkv;
  int splits, W, nq, nkv;
  int v_wgs, v_chunks, v_units;  // the first workgroups: V, v_units units of a wave each, v_chunks per 4 positions
  int chunks, units_per_wg;      // the others: queries and keys of a row, chunks each
  int q_past;                    // queries are stored past the caches
  int64_t slice;
  const uint16_t *q_norm, *k_norm, *v_norm;
  float eps;
  const float* inv_freq;
  const int32_t* seq_lens;
  int pos_offset;
  const int32_t* block_table;
  int max_pages, page;
  uint8_t *k_pool, *v_pool;
  uint32_t *k_sb, *v_sb;
  uint16_t* q_out;
  const float* x_ssq;
  int x_tiles;
  float x_k, x_eps;
};

// 8 dims of a head of a row: the sum of the projection's slices, or its bf16 values
template <int HD, bool F32>
struct Row8;
template <int HD>
struct Row8<HD, false> {
  u32x4 r;
  __device__ __forceinline__ void load(const Kv4Append& a, int row, int head, int sub) {
    const int64_t off = ((int64_t)row * (a.nq + 2 * a.nkv) + head) * HD + sub * 8;
    r = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(a.qkv) + off);
  }
  template <typename T>
  __device__ __forceinline__ void values(float, T (&v)[8]) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = (T)bits_f32(r[e] << 16);
      v[2 * e + 1] = (T)bits_f32(r[e] & 0xffff0000u);
    }
  }
};
template <int HD>
struct Row8<HD, true> {
  double s[8];
  __device__ __forceinline__ void load(const Kv4Append& a, int row, int head, int sub) {
    const float* src = reinterpret_cast<const float*>(a.qkv) + ((int64_t)row * (a.nq + 2 * a.nkv) + head) * HD + sub * 8;
    f32x4 x = *reinterpret_cast<const f32x4*>(src), y = *reinterpret_cast<const f32x4*>(src + 4);
#pragma unroll
    for (int e = 0; e < 8; ++e) s[e] = (double)(e < 4 ? x[e % 4] : y[e % 4]);
    for (int sp = 1; sp < a.splits; ++sp) {
      x = *reinterpret_cast<const f32x4*>(src + sp * a.slice);
      y = *reinterpret_cast<const f32x4*>(src + sp * a.slice + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) s[e] += (double)(e < 4 ? x[e % 4] : y[e % 4]);
    }
  }
  template <typename T>
  __device__ __forceinline__ void values(float scale, T (&v)[8]) const {  // times the row scale
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (T)(s[e] * (double)scale);
  }
};
template <int L, typename T>
__device__ __forceinline__ T lanes_sum(T x) {
#pragma unroll
  for (int o = 1; o < L; o <<= 1) x += __shfl_xor(x, o, 64);
  return x;
}
// the row scale of a projection whose input is normed later: L lanes (each with its number sub) for one row
template <int L>
__device__ __forceinline__ float row_scale(const Kv4Append& a, int row, int sub) {
  float ss = 0.0f;
  for (int j = sub; j < a.x_tiles; j += L) ss += a.x_ssq[(int64_t)row * a.x_tiles + j];
  return rsqrtf(lanes_sum<L>(ss) / a.x_k + a.x_eps);
}
// v * rsqrt(mean(v^2) + eps) * w of a head in HD / 8 lanes
template <int HD, typename T>
__device__ __forceinline__ void norm8(const Kv4Append& a, const uint16_t* w, int sub, T (&v)[8]) {
  T ss = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss += v[e] * v[e];
  ss = lanes_sum<HD / 8>(ss);
  if (!w) return;
  T r;
  if constexpr (sizeof(T) == 8) r = rsqrt(ss * (1.0 / HD) + (double)a.eps);
  else r = rsqrtf(ss / (float)HD + a.eps);
  const u32x4 g = *reinterpret_cast<const u32x4*>(w + sub * 8);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[2 * e] = v[2 * e] * r * (T)bits_f32(g[e] << 16);
    v[2 * e + 1] = v[2 * e + 1] * r * (T)bits_f32(g[e] & 0xffff0000u);
  }
}
// to bf16 by way of float32, as a cache's words are formed from float32 rows (the compiler would round once)
template <typename T>
__device__ __forceinline__ uint16_t round16(T x) {
  float f = (float)x;
  asm("" : "+v"(f));
  return f32_to_bf16(f);
}
// the codes of 8 dims, half byte e dim e, and the scale and offset of their 64 (8 lanes; every lane runs this)
template <typename T>
__device__ __forceinline__ uint32_t codes8(const T (&v)[8], uint32_t& sb) {
  T lo = v[0], hi = v[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) {
    lo = fmin(lo, v[e]);
    hi = fmax(hi, v[e]);
  }
#pragma unroll
  for (int m = 1; m < 8; m <<= 1) {
    lo = fmin(lo, __shfl_xor(lo, m, 64));
    hi = fmax(hi, __shfl_xor(hi, m, 64));
  }
  uint16_t s16 = round16(sizeof(T) == 8 ? (hi - lo) * (T)(1.0 / 15.0) : (hi - lo) / (T)15);
  if (!(bf16_to_f32(s16) > 0.0f)) s16 = 0x3f80;
  const uint16_t b16 = round16(lo);
  const T s = (T)bf16_to_f32(s16), b = (T)bf16_to_f32(b16);
  sb = (uint32_t)s16 | ((uint32_t)b16 << 16);
  // 64 bits: a product with the reciprocal, off by 2^-47 (one step from a float32 one; of 15 steps: 1e-13)
  const T r0 = (T)(1.0f / (float)s), inv = r0 * ((T)2 - s * r0);
  uint32_t cw = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    T q;
    if constexpr (sizeof(T) == 8) q = rint((v[e] - b) * inv);
    else q = rintf((v[e] - b) / s);
    cw |= (uint32_t)(int)fmin(fmax(q, (T)0), (T)15) << (4 * e);
  }
  return cw;
}

// V of 4 positions (a multiple of 4 and the next) of row b: a wave has NT of them side by side, L lanes each,
// so that bytes of neighbouring tokens, which lie together, are written as words (2048 tokens, 8 heads of 128 with
// 32 query heads: 19 us with queries and keys when V went byte by byte, 14.5 so). Other tokens stay as they are.
template <int HD, bool F32>
__device__ __forceinline__ void append_v(const Kv4Append& a, int wg) {
  using T = std::conditional_t<F32, double, float>;
  constexpr int L = HD / 8, NT = 64 / L, kParts = 4 / NT;  // a head's 4 tokens take kParts units of a wave
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, sub = lane % L, t = lane / L;
  const int quads = (a.W + 6) / 4, group = wg / a.v_chunks, chunk = wg - group * a.v_chunks;
  const int b = group / quads;
  const int64_t start = (int64_t)a.seq_lens[b] + a.pos_offset, base = (start & ~(int64_t)3) + 4 * (group - b * quads);
  const int u1 = min(a.nkv * kParts, (chunk + 1) * a.v_units);
  int last = -1;
  float scale = 1.0f;
  for (int u = chunk * a.v_units + wv; u < u1; u += 4) {
    const int head = u / kParts, t0 = (u % kParts) * NT;
    const int64_t pos64 = base + t0 + t;
    const bool stored = pos64 >= start && pos64 < start + a.W && pos64 >= 0 && pos64 < (int64_t)a.max_pages * a.page;
    const int row = b * a.W + (int)min(max(pos64 - start, (int64_t)0), (int64_t)a.W - 1), pos = stored ? (int)pos64 : 0;
    Row8<HD, F32> x;
    x.load(a, row, a.nq + a.nkv + head, sub);
    if (F32 && a.x_ssq && row != last) scale = row_scale<L>(a, row, sub);
    last = row;
    T v[8];
    x.values(scale, v);
    norm8<HD>(a, a.v_norm, sub, v);
    uint32_t sb;
    const uint32_t cw = codes8(v, sb), pw = __shfl_xor(cw, 2, 64);  // the dims 16 on (or back): the other half bytes
    const int64_t head_page = (int64_t)a.block_table[(int64_t)b * a.max_pages + pos / a.page] * a.nkv + head;
    const int slot = pos % a.page;
    // of 8 dims and the 8 that share their bytes, this lane has four bytes and the other lane four
    const bool upper = sub & 2;
    const uint32_t low = (upper ? pw >> 16 : cw) & 0xffffu, high = (upper ? cw >> 16 : pw) & 0xffffu;
    uint32_t bytes = 0;  // of dims d0 .. d0 + 3
#pragma unroll
    for (int e = 0; e < 4; ++e) bytes |= (((low >> (4 * e)) & 15u) | (((high >> (4 * e)) & 15u) << 4)) << (8 * e);
    const int d0 = (upper ? sub - 2 : sub) * 8 + (upper ? 4 : 0);
    uint32_t of[NT];  // the tokens' bytes
#pragma unroll
    for (int x = 0; x < NT; ++x) of[x] = __shfl(bytes, sub + L * x, 64);
    uint8_t* dst = a.v_pool + head_page * a.page * (HD / 2);
    if (__all(stored)) {
      // token x of this wave, dims d0 + 4 / NT * t ..: lane t has them of all its tokens
#pragma unroll
      for (int i = 0; i < 4 / NT; ++i) {
        const int e = 4 / NT * t + i;
        uint32_t w = 0;
#pragma unroll
        for (int x = 0; x < NT; ++x) w |= ((of[x] >> (8 * e)) & 255u) << (8 * x);
        uint8_t* o = dst + kv4_v_byte(HD, slot - t, d0 + e);
        if constexpr (NT == 4) *reinterpret_cast<uint32_t*>(o) = w;
        else *reinterpret_cast<uint16_t*>(o) = (uint16_t)w;
      }
    } else if (stored) {
#pragma unroll
      for (int e = 0; e < 4; ++e) dst[kv4_v_byte(HD, slot, d0 + e)] = (uint8_t)(bytes >> (8 * e));
    }
    if (stored && sub % 8 == 0) a.v_sb[(head_page * a.page + slot) * (HD / 64) + sub / 8] = sb;
  }
}

template <int HD, bool F32>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4Append a) {
  constexpr int L = HD / 8, HPW = 64 / L;  // lanes per head, heads per unit of a wave
  __shared__ double2 cs[HD / 2];   // cosine, sine
  __shared__ float2 csf[HD / 2];
  if ((int)blockIdx.x < a.v_wgs) {
    append_v<HD, F32>(a, blockIdx.x);
    return;
  }
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), sub = lane % L;
  const int wg = blockIdx.x - a.v_wgs, row = wg / a.chunks, b = row / a.W;
  const int64_t pos64 = (int64_t)a.seq_lens[b] + row % a.W + a.pos_offset;
  const bool stored = pos64 >= 0 && pos64 < (int64_t)a.max_pages * a.page;  // beyond the row's block table: dropped
  const int pos = stored ? (int)pos64 : 0;
  const int64_t pg = a.block_table[(int64_t)b * a.max_pages + pos / a.page];
  const int slot = pos % a.page;
  const int q_units = (a.nq + HPW - 1) / HPW, units = q_units + (a.nkv + HPW - 1) / HPW;
  const int u0 = (wg - row * a.chunks) * a.units_per_wg, u1 = min(units, u0 + a.units_per_wg);
  // the head of a unit's lane, and the row's head that it reads (where heads do not fill a unit: the last one)
  auto head_of = [&](int u) { return (u < q_units ? u : u - q_units) * HPW + lane / L; };
  auto load = [&](int u, Row8<HD, F32>& x) {
    x.load(a, row, u < q_units ? min(head_of(u), a.nq - 1) : a.nq + min(head_of(u), a.nkv - 1), sub);
  };
  int u = u0 + wv;
  Row8<HD, F32> nxt;
  load(min(u, units - 1), nxt);  // in flight while the angles are reduced
  const float scale = F32 && a.x_ssq ? row_scale<64>(a, row, lane) : 1.0f;
  for (int d = threadIdx.x; d < HD / 2; d += 256) {
    cs[d] = rope_angle((double)pos64, a.inv_freq[d]);
    csf[d] = float2{(float)cs[d].x, (float)cs[d].y};
  }
  __syncthreads();
  const bool first_half = sub < L / 2;
  const int d0 = (first_half ? sub : sub - L / 2) * 8;
  for (; u < u1; u += 4) {
    const Row8<HD, F32> x = nxt;
    if (u + 4 < u1) load(u + 4, nxt);
    const int head = head_of(u);
    if (u < q_units) {
      float v[8];
      x.values(scale, v);
      norm8<HD>(a, a.q_norm, sub, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {  // dim d pairs with d + HD / 2, L / 2 lanes away
        const float partner = __shfl_xor(v[e], L / 2, 64);
        const float2 t = csf[d0 + e];
        v[e] = v[e] * t.x + (first_half ? -partner : partner) * t.y;
      }
      const u32x4 out = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
      u32x4* to = reinterpret_cast<u32x4*>(a.q_out + ((int64_t)row * a.nq + head) * HD + sub * 8);
      if (head < a.nq && a.q_past) __builtin_nontemporal_store(out, to);
      else if (head < a.nq) *to = out;
    } else {
      double v[8];
      x.values(scale, v);
      norm8<HD>(a, a.k_norm, sub, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double partner = __shfl_xor(v[e], L / 2, 64);
        const double2 t = cs[d0 + e];
        v[e] = v[e] * t.x + (first_half ? -partner : partner) * t.y;
      }
      uint32_t sb;
      const uint32_t cw = codes8(v, sb);
      if (!stored || head >= a.nkv) continue;
      const int64_t at = (pg * a.nkv + head) * a.page + slot;
      if (sub % 8 == 0) a.k_sb[at * (HD / 64) + sub / 8] = sb;
      *reinterpret_cast<uint32_t*>(a.k_pool + at * (HD / 2) + kv4_k_word(sub)) = cw;
    }
  }
}

int kv4_append(const void* qkv, int splits, int B, int W, int nq, int nkv, int hd, const uint16_t* q_norm,
               const uint16_t* k_norm, const uint16_t* v_norm, float eps, const float* inv_freq,
               const int32_t* seq_lens, int pos_offset, const int32_t* block_table, int max_pages, int page,
               void* k_pool, void* v_pool, uint32_t* k_sb, uint32_t* v_sb, uint16_t* q_out, const float* x_ssq,
               int x_tiles, float x_eps, hipStream_t st) {
  const char* who = "dsk_qkv_rope_append (4-bit KV)";
  DSK_REQUIRE(hd == 128 || hd == 256, "%s: head_dim %d not supported (128, 256)", who, hd);
  DSK_REQUIRE(page % kKv4Block == 0, "%s: page size %d is not a multiple of %d", who, page, kKv4Block);
  DSK_REQUIRE(k_sb && v_sb, "%s: needs scale/bias buffers", who);
  DSK_REQUIRE(((((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)q_norm | (uintptr_t)k_norm | (uintptr_t)v_norm) & 15) |
               (((uintptr_t)k_pool | (uintptr_t)v_pool) & 15)) == 0, "%s: pointers must be 16-byte aligned", who);
  const int64_t rows = (int64_t)B * W;
  const int per_unit = hd == 128 ? 4 : 2;  // heads of a wave
  const int64_t qk_units = ceil_div(nq, per_unit) + ceil_div(nkv, per_unit);
  DSK_REQUIRE(rows <= 0x7fffffff, "%s: %lld rows", who, (long long)rows);
  // few rows: one unit per wave, so that the chip has work; many: a workgroup per row, which finds the angles once
  // (2048 rows of 40 heads, before V went apart: 18.4 us, 20.3 with a unit per wave)
  const int units_per_wg = rows < 256 ? 4 : (int)qk_units, chunks = (int)ceil_div(qk_units, units_per_wg);
  // many rows' queries leave the L2 before they are read (2048 rows: 20.6 us kept, 19.3 past it, with the read-back;
  // followed by its attention, one row 12.8 and 12.95)
  const int q_past = rows >= 256;
  const int units = nkv * (hd / 128), v_units = rows < 256 ? 4 : units, v_chunks = (int)ceil_div(units, v_units);
  const int64_t v_wgs = (int64_t)B * ((W + 6) / 4) * v_chunks;
  DSK_REQUIRE(v_wgs + rows * chunks <= 0x7fffffff, "%s: %lld rows", who, (long long)rows);
  Kv4Append a = {qkv, splits, W, nq, nkv, (int)v_wgs, v_chunks, v_units, chunks, units_per_wg, q_past, rows * (nq + 2 * nkv) * hd,
                 q_norm, k_norm, v_norm, eps, inv_freq, seq_lens, pos_offset, block_table, max_pages, page, (uint8_t*)k_pool,
                 (uint8_t*)v_pool, k_sb, v_sb, q_out, x_ssq, x_tiles, (float)(x_tiles * 16), x_eps};
  const dim3 grid((unsigned)(v_wgs + rows * chunks)), blk(256);
  if (hd == 128) {
    if (splits) hipLaunchKernelGGL((kv4_append_kernel<128, true>), grid, blk, 0, st, a);
    else hipLaunchKernelGGL((kv4_append_kernel<128, false>), grid, blk, 0, st, a);
  } else {
    if (splits) hipLaunchKernelGGL((kv4_append_kernel<256, true>), grid, blk, 0, st, a);
    else hipLaunchKernelGGL((kv4_append_kernel<256, false>), grid, blk, 0, st, a);
  }
  DSK_LAUNCH_CHECK(who);
  return DSK_OK;
}

// ----------------------------------------------------------------------------- read back
// K and V of positions first[b] + offset + i, i < n, as bf16 rows: one workgroup per 32 positions (whole
// V blocks) of a (row, kv head), 8 dims per thread and step. A copy: bound by the bytes it writes (4-bit codes of
// 32768 tokens, 8 heads of 128: 28.8 us, 6.0 TB/s read and written; of 1027, 256 dims: 6.2 us, its chain of loads).
// The stores pass the caches by: with ordinary ones the same call took 50 us once it wrote buffers that no cache held.
struct KvRead {
  const int32_t* first;
  int offset, n, nkv;
  const int32_t* block_table;
  int max_pages, page;
  const void *k_pool, *v_pool;
  const uint32_t *k_sb, *v_sb;
  uint16_t *k_out, *v_out;
};

template <int HD, int KVT>
__global__ __launch_bounds__(256) void kv_read_kernel(KvRead a) {
  constexpr int CH = HD / 8;  // 8-dim chunks of a row
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int64_t lo = (int64_t)a.first[b] + a.offset, end = min(lo + a.n, (int64_t)a.max_pages * a.page);
  const int64_t beg = max(lo, (int64_t)0);
  if (beg >= end) return;
  const int64_t base = (beg / 32 + blockIdx.x) * 32;
  if (base >= end) return;
  auto token = [&](int64_t pos) {
    const int pg = a.block_table[(int64_t)b * a.max_pages + pos / a.page];
    return ((int64_t)pg * a.nkv + kvh) * a.page + pos % a.page;
  };
  auto out_row = [&](int64_t pos) { return (((int64_t)b * a.n + (pos - lo)) * a.nkv + kvh) * HD; };
  auto rows = [&](const void* pool, const uint32_t* sb, uint16_t* out) {
    for (int i = threadIdx.x; i < 32 * CH; i += 256) {
      const int64_t pos = base + i / CH;
      const int ch = i % CH;
      if (pos < beg || pos >= end) continue;
      const int64_t tok = token(pos);
      u32x4 w;
      if constexpr (KVT == DSK_KV_BF16) {
        w = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(pool) + tok * HD + ch * 8);
      } else if constexpr (KVT == DSK_KV_U8) {
        const uint2 r = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(pool) + tok * HD + ch * 8);
        const uint32_t z = sb[tok * (HD / 64) + ch / 8];
        const float s = bits_f32(z << 16), bi = bits_f32(z & 0xffff0000u);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t two = (e < 2 ? r.x : r.y) >> (16 * (e & 1));
          w[e] = pack_bf16x2(fmaf(s, (float)(two & 255), bi), fmaf(s, (float)((two >> 8) & 255), bi));
        }
      } else {
        w = kv4_row8(*reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint8_t*>(pool) + tok * (HD / 2) + kv4_k_word(ch)),
                     kv4_scale(sb[tok * (HD / 64) + ch / 8]));
      }
      __builtin_nontemporal_store(w, reinterpret_cast<u32x4*>(out + out_row(pos) + ch * 8));
    }
  };
  rows(a.k_pool, a.k_sb, a.k_out);
  if constexpr (KVT != DSK_KV_U4) {
    rows(a.v_pool, a.v_sb, a.v_out);
  } else {
    // a thread: 4 tokens (a word) of 8 dims and of the 8 dims 16 on, from 8 words 16 bytes apart
    const int64_t tok0 = token(base);  // the block lies in one page
    const uint8_t* blk = reinterpret_cast<const uint8_t*>(a.v_pool) + tok0 * (HD / 2);
    for (int i = threadIdx.x; i < HD / 2; i += 256) {
      const int nh = i & 1, p = (i >> 1) & 1, c = (i >> 2) % (HD / 64), q4 = (i >> 2) / (HD / 64);  // q4: tokens 4 q4 ..
      const int g = q4 % 4, u = q4 / 4;
      Kv4Scale z[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) z[r] = kv4_scale(a.v_sb[(tok0 + 4 * q4 + r) * (HD / 64) + c]);
      uint32_t lo2[8][2], hi2[8][2];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        kv4_col4(*reinterpret_cast<const uint32_t*>(blk + c * 1024 + (8 * nh + e + 16 * g) * 16 + p * 8 + u * 4), z, lo2[e], hi2[e]);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int64_t pos = base + 4 * q4 + r;
        if (pos < beg || pos >= end) continue;
        uint16_t* dst = a.v_out + out_row(pos) + c * 64 + p * 32 + nh * 8;
        const uint32_t sel = r & 1 ? 0x07060302u : 0x05040100u;
        u32x4 x, y;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          x[e] = __builtin_amdgcn_perm(lo2[2 * e + 1][r / 2], lo2[2 * e][r / 2], sel);
          y[e] = __builtin_amdgcn_perm(hi2[2 * e + 1][r / 2], hi2[2 * e][r / 2], sel);
        }
        __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(dst));
        __builtin_nontemporal_store(y, reinterpret_cast<u32x4*>(dst + 16));
      }
    }
  }
}

}  // namespace dsk

using namespace dsk;

extern "C" int dsk_kv_read(const int32_t* first, int offset, int B, int n, int nkv, int hd, const int32_t* block_table,
                           int max_pages, int page, int kv_dtype, const void* k_pool, const void* v_pool,
                           const uint32_t* k_sb, const uint32_t* v_sb, uint16_t* k_out, uint16_t* v_out,
                           dsk_stream_t stream) {
  const char* who = "dsk_kv_read";
  DSK_REQUIRE(first && block_table && k_pool && v_pool && k_out && v_out, "%s: null pointer", who);
  DSK_REQUIRE(kv_dtype == DSK_KV_BF16 || kv_dtype == DSK_KV_U8 || kv_dtype == DSK_KV_U4, "%s: kv_dtype %d", who, kv_dtype);
  DSK_REQUIRE(hd == 128 || hd == 256 || (hd == 512 && kv_dtype != DSK_KV_U4),
              "%s: head_dim %d not supported (128, 256; 512 without 4-bit codes)", who, hd);
  DSK_REQUIRE(B > 0 && B <= 65535 && n > 0 && nkv > 0 && nkv <= 65535, "%s: bad shape", who);
  DSK_REQUIRE(page > 0 && max_pages > 0, "%s: bad page geometry", who);
  DSK_REQUIRE(kv_dtype != DSK_KV_U4 || page % kKv4Block == 0, "%s: 4-bit pages are multiples of %d tokens (got %d)", who,
              kKv4Block, page);
  DSK_REQUIRE(kv_dtype == DSK_KV_BF16 || (k_sb && v_sb), "%s: quantised KV needs scale/bias buffers", who);
  DSK_REQUIRE((((uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)k_out | (uintptr_t)v_out) & 15) == 0,
              "%s: pools and outputs must be 16-byte aligned", who);
  const KvRead a = {first, offset, n, nkv, block_table, max_pages, page, k_pool, v_pool, k_sb, v_sb, k_out, v_out};
  const dim3 grid((unsigned)(((int64_t)n + 62) / 32), (unsigned)nkv, (unsigned)B), blk(256);
#define DSK_READ(HDV, KVT) hipLaunchKernelGGL((kv_read_kernel<HDV, KVT>), grid, blk, 0, as_stream(stream), a)
#define DSK_READ_HD(HDV)                                     \
  if (kv_dtype == DSK_KV_BF16) DSK_READ(HDV, DSK_KV_BF16);   \
  else if (kv_dtype == DSK_KV_U8) DSK_READ(HDV, DSK_KV_U8);  \
  else DSK_READ(HDV == 512 ? 256 : HDV, DSK_KV_U4)
  if (hd == 128) {
    DSK_READ_HD(128);
  } else if (hd == 256) {
    DSK_READ_HD(256);
  } else if (kv_dtype == DSK_KV_BF16) {
    DSK_READ(512, DSK_KV_BF16);
  } else {
    DSK_READ(512, DSK_KV_U8);
  }
#undef DSK_READ_HD
#undef DSK_READ
  DSK_LAUNCH_CHECK(who);
  return DSK_OK;
}
