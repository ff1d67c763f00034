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
// One workgroup per token row and chunk of heads: the row's HD / 2 sines and cosines are found once, one
// per thread, for all heads of the chunk; then 8 dims per lane, HD / 8 lanes per head.

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
  int splits, W, nq, nkv, heads_per_wg;
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

template <int HD, bool F32>
__global__ __launch_bounds__(256) void kv4_append_kernel(Kv4Append a) {
  constexpr int L = HD / 8, HPW = 64 / L;  // lanes per head, heads per wave
  __shared__ float2 cs[HD / 2];
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, sub = lane % L;
  const int row = blockIdx.x, b = row / a.W, nheads = a.nq + 2 * a.nkv;
  const int64_t pos64 = (int64_t)a.seq_lens[b] + row % a.W + a.pos_offset;
  const bool stored = pos64 >= 0 && pos64 < (int64_t)a.max_pages * a.page;  // beyond the row's block table: dropped
  const int pos = stored ? (int)pos64 : 0;
  const int64_t pg = a.block_table[(int64_t)b * a.max_pages + pos / a.page];
  const int slot = pos % a.page;

  // the sum of the projection's slices (slice order) of 8 dims of a head, or its bf16 row
  auto load = [&](int head, float (&v)[8]) {
    const int64_t off = ((int64_t)row * nheads + min(head, nheads - 1)) * HD + sub * 8;
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
  };
  const int h0 = blockIdx.y * a.heads_per_wg, h1 = min(nheads, h0 + a.heads_per_wg);
  int head = h0 + wv * HPW + lane / L;
  float nxt[8];
  load(head, nxt);  // in flight while the angles are reduced
  float scale = 1.0f;
  if (F32 && a.x_ssq) {  // a projection whose input is normed later: its row scale
    float ss = 0.0f;
    for (int j = lane; j < a.x_tiles; j += 64) ss += a.x_ssq[(int64_t)row * a.x_tiles + j];
    scale = rsqrtf(wave_sum(ss) / a.x_k + a.x_eps);
  }
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
    if (head - lane / L + 4 * HPW < h1) load(head + 4 * HPW, nxt);
    const bool is_q = head < a.nq, is_k = !is_q && head < a.nq + a.nkv;
    const uint16_t* nw = is_q ? a.q_norm : (is_k ? a.k_norm : a.v_norm);
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss += v[e] * v[e];
    ss = row_sum<L>(ss);
    if (nw) {
      const float r = rsqrtf(ss / (float)HD + a.eps);
      const u32x4 g = *reinterpret_cast<const u32x4*>(nw + sub * 8);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[2 * e] = v[2 * e] * r * bits_f32(g[e] << 16);
        v[2 * e + 1] = v[2 * e + 1] * r * bits_f32(g[e] & 0xffff0000u);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {  // dim d pairs with d + HD / 2, L / 2 lanes away
#pragma clang fp contract(off)
      const float partner = __shfl_xor(v[e], L / 2, 64);
      const float2 t = cs[d0 + e];
      const float x = v[e] * t.x, y = partner * t.y;
      const float z = first_half ? x - y : x + y;
      if (is_q || is_k) v[e] = z;
    }
    if (is_q) {
      if (head < h1)
        *reinterpret_cast<u32x4*>(a.q_out + ((int64_t)row * a.nq + head) * HD + sub * 8) =
            u32x4{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
    }
    // codes of a group of 64 dims (8 lanes); a wave may hold query and K heads, so every lane runs them
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
    uint32_t cw = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      cw |= (uint32_t)(int)fminf(fmaxf(rintf((v[e] - bf) / sf), 0.0f), 15.0f) << (4 * e);
    const uint32_t pw = __shfl_xor(cw, 2, 64);  // the dims 16 on (or back): the other half bytes of V
    if (is_q || !stored || head >= h1) continue;
    const int64_t head_page = pg * a.nkv + (is_k ? head - a.nq : head - a.nq - a.nkv);
    if (sub % 8 == 0)
      (is_k ? a.k_sb : a.v_sb)[(head_page * a.page + slot) * (HD / 64) + sub / 8] = (uint32_t)s16 | ((uint32_t)b16 << 16);
    if (is_k) {
      *reinterpret_cast<uint32_t*>(a.k_pool + (head_page * a.page + slot) * (HD / 2) + kv4_k_word(sub)) = cw;
    } else {
      // of 8 dims and the 8 that share their bytes, this lane writes four bytes and the other lane four
      const bool upper = sub & 2;
      const uint32_t low = (upper ? pw >> 16 : cw), high = (upper ? cw >> 16 : pw);
      uint8_t* dst = a.v_pool + head_page * a.page * (HD / 2) + kv4_v_byte(HD, slot, (upper ? sub - 2 : sub) * 8) + (upper ? 64 : 0);
#pragma unroll
      for (int e = 0; e < 4; ++e) dst[16 * e] = (uint8_t)(((low >> (4 * e)) & 15) | (((high >> (4 * e)) & 15) << 4));
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
  const int heads = nq + 2 * nkv, per = hd == 128 ? 16 : 8;  // heads of one pass of a workgroup's four waves
  DSK_REQUIRE(rows <= 0x7fffffff, "%s: %lld rows", who, (long long)rows);
  // few rows: a workgroup per 16 (8) heads, so that the chip has work; many: one per row
  const int chunks = rows < 256 ? (int)ceil_div(heads, per) : 1;
  Kv4Append a = {qkv, splits, W, nq, nkv, (int)ceil_div(ceil_div(heads, chunks), per) * per, rows * heads * hd, q_norm, k_norm, v_norm, eps,
                 inv_freq, seq_lens, pos_offset, block_table, max_pages, page, (uint8_t*)k_pool, (uint8_t*)v_pool,
                 k_sb, v_sb, q_out, x_ssq, x_tiles, (float)(x_tiles * 16), x_eps};
  const dim3 grid((unsigned)rows, (unsigned)ceil_div(heads, a.heads_per_wg)), blk(256);
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
