// A 4-bit paged KV cache written as the projection's rows are formed, and the read-back of any cache.
#include "common.h"
#include "kv4.h"
#include "kv4_entry.h"
#include "kvrow.h"

namespace dsk {

// ----------------------------------------------------------------------------- append
// q, k: x * rsqrt(mean(x^2) + eps) * w, rotated by pos * inv_freq; k and v to 4-bit codes (kv4.h). A
// row stays float32 from its projection's sum to its code or its bf16 query: a rounding in between
// would move about one code in a hundred.
//
// Queries and keys: one workgroup per token row and chunk of heads; the row's HD / 2 sines and cosines are found
// once, one per thread, for all heads of the chunk; then 8 dims per lane, HD / 8 lanes per head. V, in the same
// launch: one workgroup per 4 positions.

// sin and cos of the exact product p f (a float32 angle is off by up to 2^-25 of itself: 0.004 rad at
// position 131072). Reduction by multiples k of pi/2 = P1 + P2 + P3: p f = a + (its fma remainder); a - k P1
// is exact below 2^20 (both are multiples of 2^-23, the difference below 2), the rest is carried as a second
// term through the Taylor polynomials on [-pi/4, pi/4] (their next terms are below 2^-28). Off by at most
// 4.6e-8 over 2e7 positions below 2^20, 2.5 % of the results not the nearest float32.
__device__ __forceinline__ void rope_exact(float p, float f, float& sn, float& cs) {
  const float a = p * f, alo = __builtin_fmaf(p, f, -a);
  if (fabsf(a) >= 1048576.0f) {
    sincosf(a, &sn, &cs);
    const float s0 = sn, one = 1.0f - 0.5f * alo * alo;
    sn = s0 * one + cs * alo;
    cs = cs * one - s0 * alo;
    return;
  }
  const float P1 = 1.57079637e+0f, P2 = -4.37113883e-8f, P3 = -1.71512451e-15f;
  const float k = rintf(a * 0.636619772f);
  const float r1 = __builtin_fmaf(-k, P1, a), r2 = __builtin_fmaf(-k, P2, r1);
  const float e = __builtin_fmaf(-k, P3, __builtin_fmaf(-k, P2, r1 - r2) + alo);
  const float r = r2 + e, rl = fabsf(r2) >= fabsf(e) ? (r2 - r) + e : (e - r) + r2;
  const float z = r * r, hz = 0.5f * z, w = 1.0f - hz;
  const float ps = __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, 2.75573192e-6f, -1.98412698e-4f), 8.33333333e-3f), -1.66666667e-1f);
  const float pc = __builtin_fmaf(z, __builtin_fmaf(z, __builtin_fmaf(z, -2.75573192e-7f, 2.48015873e-5f), -1.38888889e-3f), 4.16666667e-2f);
  const float s = r + __builtin_fmaf(r * z, ps, rl * w);
  const float c = w + (((1.0f - w) - hz) + __builtin_fmaf(z * z, pc, -r * rl));
  const int q = (int)k;
  const float u = q & 1 ? c : s, v = q & 1 ? s : c;
  sn = q & 2 ? -u : u;
  cs = (q + 1) & 2 ? -v : v;
}

struct Kv4Append {
  const void* qkv;
  int splits, W, nq, nkv;
  int v_wgs, v_chunks, v_units;  // the first workgroups: V, v_units units of a wave each, v_chunks per 4 positions
  int chunks, heads_per_wg;      // the others: queries and keys of a row
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

// 8 dims of a head of a row: the sum of the projection's slices (slice order), or its bf16 values
template <int HD, bool F32>
__device__ __forceinline__ void load8(const Kv4Append& a, int row, int head, int sub, float (&v)[8]) {
  const int64_t off = ((int64_t)row * (a.nq + 2 * a.nkv) + head) * HD + sub * 8;
  if constexpr (!F32) {
    const u32x4 r = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(a.qkv) + off);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[2 * e] = bits_f32(r[e] << 16);
      v[2 * e + 1] = bits_f32(r[e] & 0xffff0000u);
    }
  } else {
    const float* src = reinterpret_cast<const float*>(a.qkv) + off;
    f32x4 s0 = *reinterpret_cast<const f32x4*>(src), s1 = *reinterpret_cast<const f32x4*>(src + 4);
    for (int sp = 1; sp < a.splits; ++sp) {
      s0 += *reinterpret_cast<const f32x4*>(src + sp * a.slice);
      s1 += *reinterpret_cast<const f32x4*>(src + sp * a.slice + 4);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = s0[e];
      v[4 + e] = s1[e];
    }
  }
}
// the row scale of a projection whose input is normed later: L lanes (each with its number sub) for one row
template <int L>
__device__ __forceinline__ float row_scale(const Kv4Append& a, int row, int sub) {
  float ss = 0.0f;
  for (int j = sub; j < a.x_tiles; j += L) ss += a.x_ssq[(int64_t)row * a.x_tiles + j];
  return rsqrtf(row_sum<L>(ss) / a.x_k + a.x_eps);
}
// v * rsqrt(mean(v^2) + eps) * w of a head in HD / 8 lanes
template <int HD>
__device__ __forceinline__ void norm8(const Kv4Append& a, const uint16_t* w, int sub, float (&v)[8]) {
  float ss = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss += v[e] * v[e];
  ss = row_sum<HD / 8>(ss);
  if (!w) return;
  const float r = rsqrtf(ss / (float)HD + a.eps);
  const u32x4 g = *reinterpret_cast<const u32x4*>(w + sub * 8);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[2 * e] = v[2 * e] * r * bits_f32(g[e] << 16);
    v[2 * e + 1] = v[2 * e + 1] * r * bits_f32(g[e] & 0xffff0000u);
  }
}
// the codes of 8 dims, half byte e dim e, and the scale and offset of their 64 (8 lanes; every lane runs this)
__device__ __forceinline__ uint32_t codes8(const float (&v)[8], uint32_t& sb) {
  float lo = v[0], hi = v[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) {
    lo = fminf(lo, v[e]);
    hi = fmaxf(hi, v[e]);
  }
#pragma unroll
  for (int m = 1; m < 8; m <<= 1) {
    lo = fminf(lo, __shfl_xor(lo, m, 64));
    hi = fmaxf(hi, __shfl_xor(hi, m, 64));
  }
  uint16_t s16 = f32_to_bf16((hi - lo) / 15.0f);
  if (!(bf16_to_f32(s16) > 0.0f)) s16 = 0x3f80;
  const uint16_t b16 = f32_to_bf16(lo);
  const float sf = bf16_to_f32(s16), bf = bf16_to_f32(b16);
  sb = (uint32_t)s16 | ((uint32_t)b16 << 16);
  uint32_t cw = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) cw |= (uint32_t)(int)fminf(fmaxf(rintf((v[e] - bf) / sf), 0.0f), 15.0f) << (4 * e);
  return cw;
}

// V of 4 positions (a multiple of 4 and the next) of row b: a wave has NT of them side by side, L lanes each,
// so that bytes of neighbouring tokens, which lie together, are written as words (2048 tokens, 8 heads of 128 with
// 32 query heads: 19 us with queries, keys and values a byte at a time, 14.5 so). Other tokens stay as they are.
template <int HD, bool F32>
__device__ __forceinline__ void append_v(const Kv4Append& a, int wg) {
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
    float v[8];
    load8<HD, F32>(a, row, a.nq + a.nkv + head, sub, v);
    if (F32 && a.x_ssq) {
      if (row != last) scale = row_scale<L>(a, row, sub);
      last = row;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= scale;
    }
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
  constexpr int L = HD / 8, HPW = 64 / L;  // lanes per head, heads per wave
  __shared__ float2 cs[HD / 2];
  if ((int)blockIdx.x < a.v_wgs) {
    append_v<HD, F32>(a, blockIdx.x);
    return;
  }
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, sub = lane % L;
  const int wg = blockIdx.x - a.v_wgs, row = wg / a.chunks, b = row / a.W, nheads = a.nq + a.nkv;
  const int64_t pos64 = (int64_t)a.seq_lens[b] + row % a.W + a.pos_offset;
  const bool stored = pos64 >= 0 && pos64 < (int64_t)a.max_pages * a.page;  // beyond the row's block table: dropped
  const int pos = stored ? (int)pos64 : 0;
  const int64_t pg = a.block_table[(int64_t)b * a.max_pages + pos / a.page];
  const int slot = pos % a.page;
  const int h0 = (wg - row * a.chunks) * a.heads_per_wg, h1 = min(nheads, h0 + a.heads_per_wg);
  int head = h0 + wv * HPW + lane / L;
  float nxt[8];
  load8<HD, F32>(a, row, min(head, nheads - 1), sub, nxt);  // in flight while the angles are reduced
  const float scale = F32 && a.x_ssq ? row_scale<64>(a, row, lane) : 1.0f;
  for (int d = threadIdx.x; d < HD / 2; d += 256) {
    float sn, c;
    rope_exact((float)pos64, a.inv_freq[d], sn, c);
    cs[d] = float2{c, sn};
  }
  __syncthreads();
  const bool first_half = sub < L / 2;
  const int d0 = (first_half ? sub : sub - L / 2) * 8;
  for (; head - lane / L < h1; head += 4 * HPW) {  // whole waves: the shuffles below need every lane
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = nxt[e] * scale;
    if (head - lane / L + 4 * HPW < h1) load8<HD, F32>(a, row, min(head + 4 * HPW, nheads - 1), sub, nxt);
    const bool is_q = head < a.nq;
    norm8<HD>(a, is_q ? a.q_norm : a.k_norm, sub, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) {  // dim d pairs with d + HD / 2, L / 2 lanes away
#pragma clang fp contract(off)
      const float partner = __shfl_xor(v[e], L / 2, 64);
      const float2 t = cs[d0 + e];
      const float x = v[e] * t.x, y = partner * t.y;
      v[e] = first_half ? x - y : x + y;
    }
    if (is_q && head < h1)
      *reinterpret_cast<u32x4*>(a.q_out + ((int64_t)row * a.nq + head) * HD + sub * 8) =
          u32x4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
    if (__all(is_q)) continue;
    uint32_t sb;
    const uint32_t cw = codes8(v, sb);  // a wave may hold query and K heads, so every lane runs it
    if (is_q || !stored || head >= h1) continue;
    const int64_t at = (pg * a.nkv + head - a.nq) * a.page + slot;
    if (sub % 8 == 0) a.k_sb[at * (HD / 64) + sub / 8] = sb;
    *reinterpret_cast<uint32_t*>(a.k_pool + at * (HD / 2) + kv4_k_word(sub)) = cw;
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
  const int heads = nq + nkv, per = hd == 128 ? 16 : 8;  // query and K heads of one pass of a workgroup's four waves
  DSK_REQUIRE(rows <= 0x7fffffff, "%s: %lld rows", who, (long long)rows);
  // few rows: a workgroup per 16 (8) heads, so that the chip has work; many: one per row
  const int heads_per_wg = rows < 256 ? per : (int)ceil_div(heads, per) * per, chunks = (int)ceil_div(heads, heads_per_wg);
  const int units = nkv * (hd / 128), v_units = rows < 256 ? 4 : units, v_chunks = (int)ceil_div(units, v_units);
  const int64_t v_wgs = (int64_t)B * ((W + 6) / 4) * v_chunks;
  DSK_REQUIRE(v_wgs + rows * chunks <= 0x7fffffff, "%s: %lld rows", who, (long long)rows);
  Kv4Append a = {qkv, splits, W, nq, nkv, (int)v_wgs, v_chunks, v_units, chunks, heads_per_wg, rows * (nq + 2 * nkv) * hd,
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
// V blocks) of a (row, kv head), 8 dims per thread and step. A copy: bound by the bytes it writes.
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
      *reinterpret_cast<u32x4*>(out + out_row(pos) + ch * 8) = w;
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
        *reinterpret_cast<u32x4*>(dst) = x;
        *reinterpret_cast<u32x4*>(dst + 16) = y;
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
