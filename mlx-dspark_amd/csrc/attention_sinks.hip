// Attention over a paged KV cache of bf16, 8-bit or 4-bit values with an optional sliding window and the
// context's first tokens (sinks) visible beside it: decode, verify and prompt passes.
//
// Transposed as the other attention kernels are, S^T[key][q] = K . Q^T and O^T[d][q] = V^T . P^T, so a lane
// owns one query column: lane l (n = l % 16, g = l / 16) holds query n's scores of keys 4 g + r and
// 16 + 4 g + r of a 32-key block, which are its 8 items of the P operand, and V^T comes in that key order.
// Keys are visited in aligned blocks of 32: first the blocks that hold sinks, then those from the window's
// start (or 0) to the last key. Scores, running maximum, sum and output are float32; a probability enters
// the P.V product as three bf16 terms (within 2^-26 of it), in passes of many rows also as two (2^-17), as the
// caller says: two moved the logits of small models to twice the distance that float32 orders of summation
// alone move them by, three left them there; they cost a prompt of 4096 tokens a fifth (316 us, 250 with two),
// one of 2048 under a window of 1024 a tenth (101, 91), decoding 9 %.
//
// The maximum moves only when a score passes it by 2^8: below that the exponentials stay in float32's
// range and nothing is lost, and a block costs one vote instead of two lane exchanges and a rescale.
//
// Measured, us (the kernel, then with the join of its splits in a graph; rates are of the whole):
//   4-bit, 32 heads of 128 over 8: one token after 16384 .. 65536 in 4 rows 43, 51: 3.4 TB/s of codes; 16 tokens
//     after 4096 11.7, 15.5; a prompt of 4096 tokens 268, unsplit: 0.51 PFLOP/s of scores and outputs, 1.03 with the
//     three terms
//   8-bit, window 4096 and 64 sinks, one token in 8 rows of 2048 .. 32768 19, 23.7: 2.8 TB/s
//   bf16, 16 heads of 256 over 8, window 1024, 9 tokens 12.7, 16
//   4-bit, the same window, a prompt of 2048 tokens after 1000 102, unsplit: 0.34 PFLOP/s, 0.67 with the terms
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "kv4.h"

namespace dsk {

// x / d for 0 <= x < 2^31 by a multiplication (d is the same for a whole launch): a division costs a wave
// some 30 instructions, a dozen of them stood before a split's first load.
struct FastDiv {
  uint32_t d, m, s;
  __host__ explicit FastDiv(uint32_t v = 1) : d(v), s(0) {
    while ((1ull << s) < v) ++s;
    m = (uint32_t)(((1ull << 32) * ((1ull << s) - v)) / v + 1);
  }
  __device__ __forceinline__ int quot(int x) const { return (int)((__umulhi((uint32_t)x, m) + (uint32_t)x) >> s); }
};

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

struct SinkArgs {
  const uint16_t* q;  // [B*W][nq*HD]
  int B, W, nq, nkv, G, R;  // R = W * G query rows per (row b, kv head)
  float scale, softcap;
  int causal, window, sinks;  // window 0: none
  const int32_t* seq_lens;
  const int32_t* block_table;
  int max_pages, page;
  const void *k_pool, *v_pool;
  const uint32_t *k_sb, *v_sb;
  uint16_t* out;
  int out_packed;
  int groups;    // row groups of a (row b, kv head), one workgroup each per split
  int grows;     // rows per group
  int slots;     // splits on the grid per kv head: placed by the rows' lengths (balanced), or nsplit for each row
  int nsplit, balanced;
  float* part_o;   // [slot][kv head][R][HD] unnormalised outputs
  float* part_ml;  // [slot][kv head][R][2] running maximum (of scores times c2) and sum
  int2* part_at;   // [row b] first slot and number of splits (balanced)
  FastDiv by_page, by_G, by_nkv, by_nsplit;
};

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kSplitUnit = 4;       // splits are multiples of this many 32-key blocks: one per wave, or two chunks of 64
constexpr float kMaxSlack = 8.0f;   // how far (log2) a score may pass the running maximum
constexpr int kDecodeMaxW = 64;      // new tokens per row of a decode or verify pass
constexpr int kSpreadRows = 5;      // query rows whose three terms fit the 16 columns of a tile
constexpr int kBalancedRows = 64;   // rows whose lengths a workgroup reads to place its split, one per lane

// The 32-key blocks that query tokens i0 .. i1 of row b look at.
struct KeyPlan {
  int off, j_beg, j_end;  // cached keys; first key of the window range, end of the keys
  int beg, nA, T;         // sink blocks 0 .. nA - 1 sit at 32 v, the others at beg + 32 (v - nA); T in all
  __device__ __forceinline__ int base(int v) const { return v < nA ? 32 * v : beg + 32 * (v - nA); }
};
__device__ __forceinline__ KeyPlan key_plan(const SinkArgs& a, int len, int i0, int i1) {
  KeyPlan p;
  p.off = max(len, 0);
  const int Lk = (int)min((int64_t)p.off + a.W, (int64_t)a.max_pages * a.page);
  const bool windowed = a.causal && a.window > 0;
  p.j_end = a.causal ? min(Lk, p.off + i1 + 1) : Lk;
  p.j_beg = windowed ? min(p.j_end, max(0, p.off + i0 - a.window + 1)) : 0;
  p.beg = p.j_beg & ~31;
  p.nA = windowed ? (min(a.sinks, p.j_end) + 31) / 32 : 0;
  if (32 * p.nA >= p.beg) p.nA = p.beg = 0;  // the two ranges meet
  p.T = p.nA + (p.j_end - p.beg + 31) / 32;
  return p;
}

// Which split a workgroup runs: the row b, its slot of the partial buffers, its blocks [v0, v1) and the
// number of splits that the row (and group) has. Balanced: blocks per split from the rows' summed lengths, so that rows
// of very different lengths load the chip evenly. live == 0: nothing to do.
struct SplitTask {
  int b, slot, v0, v1, live;
  KeyPlan p;
};
// Rows by their lengths, one row per lane (one load for all: read one after the other they cost a round trip
// each): the fewest blocks per split, in units, with which the rows' splits fit the slots, and the lane's row's
// number of splits. sum ceil(T / bps) <= sum T / bps + B gives one that fits; a few halvings from the ideal
// sum T / slots find a better one (32 rows of 4096 keys, 32 heads: 75 us with the first, 53 so).
struct Placement {
  int lens, live, bps;
};
__device__ __forceinline__ Placement placement(const SinkArgs& a) {
  const int lane = threadIdx.x & 63;
  Placement p;
  p.lens = a.seq_lens[min(lane, a.B - 1)];
  const int T = key_plan(a, p.lens, 0, a.W - 1).T;
  auto sum = [&](int x) {
    int s = 0;
    for (int b = 0; b < a.B; ++b) s += __builtin_amdgcn_readlane(x, b);
    return s;
  };
  auto units = [](int x) { return max(kSplitUnit, (x + kSplitUnit - 1) & -kSplitUnit); };
  auto splits = [&](int bps) { return max(1, (int)((uint32_t)(T + bps - 1) / (uint32_t)bps)); };
  const int total = sum(T);
  int lo = units((int)((uint32_t)(total + a.slots - 1) / (uint32_t)a.slots));
  p.bps = units((int)((uint32_t)(total + a.slots - a.B - 1) / (uint32_t)(a.slots - a.B)));
#pragma unroll 1
  for (int i = 0; i < 4 && lo < p.bps; ++i) {
    const int x = i == 0 ? lo : units((lo + p.bps) / 2 - kSplitUnit + 1);
    if (sum(splits(x)) <= a.slots) p.bps = x;
    else lo = x + kSplitUnit;
  }
  p.live = splits(p.bps);
  return p;
}
__device__ __forceinline__ int even_blocks(const SinkArgs& a, int T) {
  return max(kSplitUnit, (a.by_nsplit.quot(T + a.nsplit - 1) + kSplitUnit - 1) & -kSplitUnit);
}
__device__ __forceinline__ SplitTask split_task(const SinkArgs& a, int slot, int group) {
  SplitTask t;
  t.slot = slot;
  t.live = 0;
  if (a.balanced) {
    const Placement pl = placement(a);
    int first = 0;
    for (int b = 0; b < a.B; ++b) {
      const int live = __builtin_amdgcn_readlane(pl.live, b);
      if (slot < first + live) {
        t.b = b;
        t.p = key_plan(a, __builtin_amdgcn_readlane(pl.lens, b), 0, a.W - 1);
        t.live = live;
        t.v0 = (slot - first) * pl.bps;
        t.v1 = min(t.p.T, t.v0 + pl.bps);
        // for the join: its many workgroups would take longer to place the rows again than to read this
        if (slot == first && group == 0 && slot * a.nkv == (int)blockIdx.x && threadIdx.x == 0) a.part_at[b] = int2{first, live};
        break;
      }
      first += live;
    }
    return t;
  }
  t.b = a.by_nsplit.quot(slot);
  t.p = key_plan(a, a.seq_lens[t.b], a.by_G.quot(group * a.grows), a.by_G.quot(min(a.R, (group + 1) * a.grows) - 1));
  const int bps = even_blocks(a, t.p.T);
  const int s = slot - t.b * a.nsplit, live = max(1, (t.p.T + bps - 1) / bps);
  if (s < live) t.live = live;
  t.v0 = s * bps;
  t.v1 = min(t.p.T, t.v0 + bps);
  return t;
}

// The keys a query at position pos sees: j <= last and (j >= first or j < sinks). Selects throughout: with
// branches here the compiler has dropped the masking of a score in a branch's far side.
struct Sight {
  int first, last, sinks;
  __device__ __forceinline__ bool sees(int j) const { return bool((int)(j <= last) & ((int)(j >= first) | (int)(j < sinks))); }
};
__device__ __forceinline__ Sight sight(const SinkArgs& a, const KeyPlan& p, int pos) {
  const bool windowed = a.causal && a.window > 0;
  return Sight{windowed ? pos - a.window + 1 : 0, a.causal ? min(p.j_end - 1, pos) : p.j_end - 1, windowed ? a.sinks : 0};
}
// whether block [j, j + 31] needs no mask for queries at positions lo .. hi, and whether none of them sees it
__device__ __forceinline__ bool block_open(const SinkArgs& a, const KeyPlan& p, int j, int lo, int hi) {
  if (j + 31 >= p.j_end) return false;
  if (!a.causal) return true;
  return j + 31 <= lo && (a.window <= 0 || j > hi - a.window || j + 31 < a.sinks);
}
__device__ __forceinline__ bool block_shut(const SinkArgs& a, int j, int lo, int hi) {
  return a.causal && (j > hi || (a.window > 0 && j + 31 <= lo - a.window && j >= a.sinks));
}
// whether no query of the plan sees key j: what stands there (the slots behind the last key, expired keys)
// is kept out of the P.V product, where a probability of 0 would not undo an infinity or a NaN
__device__ __forceinline__ bool key_dead(const SinkArgs& a, const KeyPlan& p, int j) {
  return bool((int)(j >= p.j_end) | ((int)(j < p.j_beg) & (int)(j >= a.sinks)));
}

__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ bool nonfinite2(uint32_t w) {
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}
// whether 4-bit values under this scale and offset may leave what kv4_scale takes, or the largest float
__device__ __forceinline__ bool wide2(uint32_t sb) {
  return (sb & 0x7f80u) >= 0x7300u || (sb & 0x7f800000u) >= 0x7d000000u;  // s >= 2^103, |b| >= 2^123
}
// Parts pass the L2 by: the join's workgroups run on other dies (12 tokens after 8192, 32 heads: 18.1 us with
// ordinary stores, 17.7 so; 16 heads of 256: 26.3 and 25.2).
__device__ __forceinline__ void store_part(float* to, f32x4 x) { __builtin_nontemporal_store(x, reinterpret_cast<f32x4*>(to)); }
__device__ __forceinline__ int64_t sink_out_index(const SinkArgs& a, int HD, int b, int r, int kvh, int d) {
  const int i = a.by_G.quot(r);
  const int64_t m = (int64_t)b * a.W + i, k = (int64_t)(kvh * a.G + r - i * a.G) * HD + d;
  return a.out_packed ? apack_index(m, k, (int64_t)a.nq * HD / 64) : m * a.nq * HD + k;
}

template <int N, int I = 0, class F>
__device__ __forceinline__ void static_for(F f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    static_for<N, I + 1>(f);
  }
}

// The running state of one tile of 16 queries over the keys seen so far; a probability goes into the P.V
// products as kTerms bf16 terms.
template <int HD, int kTerms>
struct Tile {
  float m, l;  // maximum (times c2) of the lane's query; the lane's own keys' sum
  f32x4 o[HD / 16];
  __device__ __forceinline__ void clear() {
    m = -__builtin_inff();
    l = 0.0f;
#pragma unroll
    for (int d = 0; d < HD / 16; ++d) o[d] = f32x4{0, 0, 0, 0};
  }
  // the lane's largest score (times c2)
  template <int NKT>
  static __device__ __forceinline__ float largest(const f32x4 (&st)[NKT], float c2) {
    float mx = -__builtin_inff();
#pragma unroll
    for (int t = 0; t < NKT; ++t) mx = fmaxf(mx, fmaxf(fmaxf(st[t][0], st[t][1]), fmaxf(st[t][2], st[t][3])));
    return mx * c2;
  }
  // whether a score passes the running maximum by more than its slack; if so for any lane, raise() in all
  __device__ __forceinline__ bool passes(float mx) const { return mx > m + kMaxSlack; }
  __device__ __forceinline__ void raise(float mx) {
    mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
    mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
    const float mn = fmaxf(m, mx);
    const float alpha = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    l *= alpha;
#pragma unroll
    for (int d = 0; d < HD / 16; ++d) o[d] *= alpha;
  }
  // a block's scores -> probabilities in place
  __device__ __forceinline__ void soften(f32x4& a, f32x4& b, float c2) {
    const float mb = m == -__builtin_inff() ? 0.0f : m;  // a row with no visible key yet: exp2(-inf) = 0
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      a[r] = __builtin_amdgcn_exp2f(fmaf(a[r], c2, -mb));
      l += a[r];
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      b[r] = __builtin_amdgcn_exp2f(fmaf(b[r], c2, -mb));
      l += b[r];
    }
  }
  // the bf16 terms of 8 probabilities (tiles t, t + 1 of a 32-key block)
  static __device__ __forceinline__ void terms(const f32x4& a, const f32x4& b, u32x4 (&t)[kTerms]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4& s = i < 2 ? a : b;
      uint32_t w[kTerms];
      split_terms_bf16x2<kTerms>(s[2 * (i & 1)], s[2 * (i & 1) + 1], w);
#pragma unroll
      for (int k = 0; k < kTerms; ++k) t[k][i] = w[k];
    }
  }
  // of 8 probabilities the term that the lane's column takes (kTerms 1): k1, k2 are 1 from the second and third on
  static __device__ __forceinline__ void own_term(const f32x4& a, const f32x4& b, float k1, float k2, u32x4& t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const f32x4& s = i < 2 ? a : b;
      float x = s[2 * (i & 1)], y = s[2 * (i & 1) + 1];
      uint32_t w = pack_bf16x2(x, y);
      x = fmaf(-k1, bits_f32(w << 16), x);
      y = fmaf(-k1, bits_f32(w & 0xffff0000u), y);
      w = pack_bf16x2(x, y);
      x = fmaf(-k2, bits_f32(w << 16), x);
      y = fmaf(-k2, bits_f32(w & 0xffff0000u), y);
      t[i] = pack_bf16x2(x, y);
    }
  }
  // O^T += V^T . P^T for d tiles D .. D + 3 and a block's 32 keys, term by term: four independent products
  // between two on the same accumulator.
  template <int D>
  __device__ __forceinline__ void add4(const u32x4 (&v)[4], const u32x4 (&t)[kTerms]) {
#pragma unroll
    for (int k = 0; k < kTerms; ++k)
#pragma unroll
      for (int d = 0; d < 4; ++d) o[D + d] = mfma16(v[d], t[k], o[D + d]);
  }
};
__device__ __forceinline__ u32x4 finite_only(u32x4 x) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const uint32_t l = (x[w] & 0x7f80u) == 0x7f80u ? 0u : 0xffffu, h = (x[w] & 0x7f800000u) == 0x7f800000u ? 0u : 0xffff0000u;
    x[w] &= l | h;
  }
  return x;
}
// the value (bf16) of dim d of V at pool token tok; apart: whether it is staged as 0
template <int HD, int KVT>
__device__ __forceinline__ uint32_t v_value(const SinkArgs& a, uint32_t tok, int d, bool& apart) {
  if constexpr (KVT == DSK_KV_BF16) {
    const uint32_t v = reinterpret_cast<const uint16_t*>(a.v_pool)[(int64_t)tok * HD + d];
    apart = (v & 0x7f80u) == 0x7f80u;
    return v;
  } else {
    const uint32_t z = a.v_sb[(int64_t)tok * (HD / 64) + d / 64];
    uint32_t c;
    if constexpr (KVT == DSK_KV_U8) {
      c = reinterpret_cast<const uint8_t*>(a.v_pool)[(int64_t)tok * HD + d];
    } else {
      const uint32_t blk = tok & ~31u;  // pages are whole blocks
      c = reinterpret_cast<const uint8_t*>(a.v_pool)[(int64_t)blk * (HD / 2) + kv4_v_byte(HD, (int)(tok - blk), d)];
      c = d & 16 ? c >> 4 : c & 15;
    }
    const uint32_t v = f32_to_bf16(fmaf(bits_f32(z << 16), (float)c, bits_f32(z & 0xffff0000u)));
    apart = KVT == DSK_KV_U4 ? wide2(z) : (v & 0x7f80u) == 0x7f80u;
    return v;
  }
}
// Infinities and NaN in V where not every query sees every key: a probability of 0 would not keep them out of a
// product (4-bit codes: all of a group whose scale or offset could reach them). Such operands are staged without them, and each is added here to the queries that see its key
// (tok: the block's first pool token). Rare, and apart from the products, which stay one run of instructions.
template <int HD, int KVT, int TPW, int TERMS>
__device__ __forceinline__ void add_nonfinite(const SinkArgs& a, Tile<HD, TERMS> (&tile)[TPW], const Sight (&see)[TPW],
                                              const u32x4 (&t)[TPW][TERMS], int base, uint32_t tok, int lane) {
#pragma unroll 1
  for (int k = 0; k < 32; ++k) {
    const int e = (k / 16) * 4 + k % 4, from = (lane & 15) + 16 * ((k % 16) / 4);
    float p[TPW];
    bool vis[TPW];
#pragma unroll
    for (int u = 0; u < TPW; ++u) {
      p[u] = 0.0f;
#pragma unroll
      for (int i = 0; i < TERMS; ++i) {
        const uint32_t w = e < 4 ? (e < 2 ? t[u][i][0] : t[u][i][1]) : (e < 6 ? t[u][i][2] : t[u][i][3]);
        p[u] += bits_f32((w << (e & 1 ? 0 : 16)) & 0xffff0000u);
      }
      vis[u] = see[u].sees(base + k);
      if constexpr (TERMS == 1) {  // the terms are in three columns: all of them to the first
        const int c = (lane & 15) % kSpreadRows + (from & 48);
        const float t0 = __shfl(p[u], c, 64), t1 = __shfl(p[u], c + kSpreadRows, 64), t2 = __shfl(p[u], c + 2 * kSpreadRows, 64);
        p[u] = t0 + t1 + t2;
        vis[u] = bool((int)vis[u] & (int)((lane & 15) < kSpreadRows));
      } else {
        p[u] = __shfl(p[u], from, 64);
      }
    }
#pragma unroll
    for (int d = 0; d < HD / 16; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        bool apart;
        const uint32_t v = v_value<HD, KVT>(a, tok + k, 16 * d + 4 * (lane >> 4) + r, apart);
#pragma unroll
        for (int u = 0; u < TPW; ++u)
          tile[u].o[d][r] = (int)apart & (int)vis[u] ? fmaf(p[u], bits_f32(v << 16), tile[u].o[d][r]) : tile[u].o[d][r];
      }
  }
}

// masks of a 32-key block's (or two blocks') scores: lane holds keys base + 16 t + 4 g + r
template <int NKT>
__device__ __forceinline__ void mask_scores(const Sight& see, f32x4 (&st)[NKT], int t0, int base, int g) {
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    f32x4 x = st[t0 + t];
    const int j = base + 16 * t + 4 * g;
    x = f32x4{see.sees(j) ? x[0] : -__builtin_inff(), see.sees(j + 1) ? x[1] : -__builtin_inff(),
              see.sees(j + 2) ? x[2] : -__builtin_inff(), see.sees(j + 3) ? x[3] : -__builtin_inff()};
    st[t0 + t] = x;
  }
}

// 4 codes of an 8-bit row -> two words of bf16(s c + b), c as a float16 denormal (kv4.h): 4.1 ns of a SIMD per
// code at two waves where v_cvt_f32_ubyte and an fma take 5.4
__device__ __forceinline__ u32x2 kv8_row4(uint32_t w, float s24, float b) {
  const uint32_t x = w & 0x00ff00ffu, y = (w >> 8) & 0x00ff00ffu;
  return u32x2{pack_bf16x2(kv4_lo(x, s24, b), kv4_lo(y, s24, b)), pack_bf16x2(kv4_hi(x, s24, b), kv4_hi(y, s24, b))};
}
__device__ __forceinline__ u32x4 kv8_row8(uint32_t w0, uint32_t w1, uint32_t z) {
  const Kv4Scale k = kv4_scale(z);
  const u32x2 a = kv8_row4(w0, k.s24, k.b), b = kv8_row4(w1, k.s24, k.b);
  return u32x4{a[0], a[1], b[0], b[1]};
}

// ----------------------------------------------------------------------------- K and V of a block
// One wave's loads of a 32-key block, kept raw until they are used (so the next block's are in flight
// meanwhile), and the operands they become.
// Every member is one load: parts of a wider load held in separate variables would be copied (and so
// waited for) where the loop comes round.
// K: u32x4 per 16-key tile and 32-dim step (A operand of the score product).
template <int HD, int KVT>
struct KRaw {
  static constexpr bool kBytes = KVT == DSK_KV_U8;
  u32x4 q[2][KVT == DSK_KV_BF16 ? HD / 32 : (kBytes ? HD / 64 : HD / 128)];
  u32x2 sb[2][KVT == DSK_KV_BF16 ? 1 : HD / 128];
  // tok: pool token of the block's first key
  __device__ __forceinline__ void load(const SinkArgs& a, uint32_t tok, int lane) {
    const int n = lane & 15, g = lane >> 4;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int64_t row = (int64_t)tok + 16 * t + n;
      if constexpr (KVT == DSK_KV_BF16) {
        const uint16_t* src = reinterpret_cast<const uint16_t*>(a.k_pool) + row * HD + 8 * g;
#pragma unroll
        for (int s = 0; s < HD / 32; ++s) q[t][s] = *reinterpret_cast<const u32x4*>(src + 32 * s);
      } else if constexpr (kBytes) {
        const uint8_t* src = reinterpret_cast<const uint8_t*>(a.k_pool) + row * HD + 16 * g;
#pragma unroll
        for (int s = 0; s < HD / 64; ++s) q[t][s] = *reinterpret_cast<const u32x4*>(src + 64 * s);
      } else {
        const uint8_t* src = reinterpret_cast<const uint8_t*>(a.k_pool) + row * (HD / 2) + 16 * g;
#pragma unroll
        for (int s = 0; s < HD / 128; ++s) q[t][s] = *reinterpret_cast<const u32x4*>(src + 64 * s);
      }
      if constexpr (KVT != DSK_KV_BF16) {
#pragma unroll
        for (int c = 0; c < HD / 128; ++c) sb[t][c] = *reinterpret_cast<const u32x2*>(a.k_sb + row * (HD / 64) + 2 * c);
      }
    }
  }
  // first of the 8 dims that step s takes from lane group g (the queries come in the same order): an 8-bit
  // row's lane holds 16 consecutive dims for two steps
  static __device__ __forceinline__ int dim(int s, int g) { return kBytes ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 32 * s + 8 * g; }
  __device__ __forceinline__ u32x4 operand(int t, int s) const {
    if constexpr (KVT == DSK_KV_BF16) return q[t][s];
    else if constexpr (kBytes) return kv8_row8(q[t][s / 2][2 * (s & 1)], q[t][s / 2][2 * (s & 1) + 1], sb[t][s / 4][(s / 2) & 1]);
    else return kv4_row8(q[t][s / 4][s % 4], kv4_scale(sb[t][s / 4][(s / 2) & 1]));
  }
};

// V operands (d tile, lane) in LDS: 16 bytes per lane, a pad after each lane group spreads the transposing
// writes of row-major caches over the banks
constexpr int kVGroup = 256 + 16, kVTile = 4 * kVGroup;  // bytes per lane group, per 16-dim tile

// 4-bit V of one 64-dim chunk c of a block: four d tiles' operands from one 16-byte load per lane
template <int HD>
struct V4Raw {
  u32x4 q;
  uint32_t sb[8];
  __device__ __forceinline__ void load(const SinkArgs& a, uint32_t tok, int c, int lane) {
    q = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint8_t*>(a.v_pool) + (int64_t)tok * (HD / 2) + c * 1024 + lane * 16);
    const uint32_t* src = a.v_sb + ((int64_t)tok + 4 * (lane >> 4)) * (HD / 64) + c;
#pragma unroll
    for (int e = 0; e < 8; ++e) sb[e] = src[(16 * (e / 4) + e % 4) * (HD / 64)];
  }
  // d tiles 4 c + 2 p + h
  __device__ __forceinline__ void operands(u32x4 (&v)[4]) const {
    Kv4Scale z[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = kv4_scale(sb[e]);
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      uint32_t lo[2][2], hi[2][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) kv4_col4(q[2 * p + u], z + 4 * u, lo[u], hi[u]);
      v[2 * p] = u32x4{lo[0][0], lo[0][1], lo[1][0], lo[1][1]};
      v[2 * p + 1] = u32x4{hi[0][0], hi[0][1], hi[1][0], hi[1][1]};
    }
  }
  // the words of keys that no query sees cleared, and the wide ones; whether there were such
  __device__ __forceinline__ bool clean(const SinkArgs& a, const KeyPlan& p, int base, int lane) {
    asm volatile("" : "+s"(base));  // keeps the tests inside the caller's branch
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      sb[e] = key_dead(a, p, base + 16 * (e / 4) + 4 * (lane >> 4) + e % 4) ? 0u : sb[e];
      bad |= wide2(sb[e]);
      sb[e] = wide2(sb[e]) ? 0u : sb[e];
    }
    return bad;
  }
};

// All of a block's 4-bit V: chunk c's 16 bytes and, per 16-key tile, the words of 4 keys
template <int HD>
struct V4Block {
  u32x4 q[HD / 64];
  u32x4 sb[2][HD / 64];  // word (r, c) of tile u: element r * (HD / 64) + c of sb[u]
  __device__ __forceinline__ void load(const SinkArgs& a, uint32_t tok, int lane) {
    const uint8_t* src = reinterpret_cast<const uint8_t*>(a.v_pool) + (int64_t)tok * (HD / 2) + lane * 16;
    const uint32_t* w = a.v_sb + ((int64_t)tok + 4 * (lane >> 4)) * (HD / 64);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int x = 0; x < HD / 64; ++x) sb[u][x] = *reinterpret_cast<const u32x4*>(w + 16 * u * (HD / 64) + 4 * x);
#pragma unroll
    for (int c = 0; c < HD / 64; ++c) q[c] = *reinterpret_cast<const u32x4*>(src + c * 1024);
  }
  __device__ __forceinline__ void pin() {  // as VRowsRaw::pin
#pragma unroll
    for (int x = 0; x < HD / 64; ++x) asm volatile("" : "+v"(q[x]), "+v"(sb[0][x]), "+v"(sb[1][x]));
  }
  __device__ __forceinline__ bool clean(const SinkArgs& a, const KeyPlan& p, int base, int lane) {  // as V4Raw::clean
    asm volatile("" : "+s"(base));
    bool bad = false;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint32_t keep = key_dead(a, p, base + 16 * u + 4 * (lane >> 4) + r) ? 0u : ~0u;
#pragma unroll
        for (int c = 0; c < HD / 64; ++c) {
          uint32_t w = sb[u][(r * (HD / 64) + c) / 4][(r * (HD / 64) + c) % 4] & keep;
          bad |= wide2(w);
          sb[u][(r * (HD / 64) + c) / 4][(r * (HD / 64) + c) % 4] = wide2(w) ? 0u : w;
        }
      }
    return bad;
  }
  // d tiles 4 c + 2 p + h
  __device__ __forceinline__ void operands(int c, u32x4 (&v)[4]) const {
    Kv4Scale z[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int x = (e % 4) * (HD / 64) + c;
      z[e] = kv4_scale(sb[e / 4][x / 4][x % 4]);
    }
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      uint32_t lo[2][2], hi[2][2];
#pragma unroll
      for (int u = 0; u < 2; ++u) kv4_col4(q[c][2 * p + u], z + 4 * u, lo[u], hi[u]);
      v[2 * p] = u32x4{lo[0][0], lo[0][1], lo[1][0], lo[1][1]};
      v[2 * p + 1] = u32x4{hi[0][0], hi[0][1], hi[1][0], hi[1][1]};
    }
  }
};

// row-major V (bf16, 8-bit): 4 keys x C dims (8, or 16 of 8 bits), transposed on their way into the operand
// order in LDS
template <int HD, int KVT, int C = 8>
struct VRowsRaw {
  static constexpr bool kBytes = KVT == DSK_KV_U8;
  static_assert(C == 8 || (kBytes && C == 16), "one 8- or 16-byte load per key");
  u32x4 q[C == 16 || !kBytes ? 4 : 1];
  u32x2 h[kBytes && C == 8 ? 4 : 1];
  uint32_t sb[4];
  // quad: keys 4 quad .. + 3 of the block, ch: dims C ch .. + C - 1
  __device__ __forceinline__ void load(const SinkArgs& a, uint32_t tok, int quad, int ch) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t row = (int64_t)tok + 4 * quad + r;
      if constexpr (!kBytes) {
        q[r] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(a.v_pool) + row * HD + 8 * ch);
      } else {
        const uint8_t* src = reinterpret_cast<const uint8_t*>(a.v_pool) + row * HD + C * ch;
        if constexpr (C == 16) q[r] = *reinterpret_cast<const u32x4*>(src);
        else h[r] = *reinterpret_cast<const u32x2*>(src);
        sb[r] = a.v_sb[row * (HD / 64) + ch / (64 / C)];
      }
    }
  }
  // not used before this point: the scheduler would otherwise turn V into operands (and wait for it) while
  // the scores are still on their way
  __device__ __forceinline__ void pin() {
    if constexpr (C == 16 || !kBytes) asm volatile("" : "+v"(q[0]), "+v"(q[1]), "+v"(q[2]), "+v"(q[3]));
    else asm volatile("" : "+v"(h[0]), "+v"(h[1]), "+v"(h[2]), "+v"(h[3]));
    if constexpr (kBytes) asm volatile("" : "+v"(sb[0]), "+v"(sb[1]), "+v"(sb[2]), "+v"(sb[3]));
  }
  // base: the block's first key; dst: the block's operands in LDS. check: without the keys that no query sees
  // and what is not finite; whether there was such
  __device__ __forceinline__ bool store(const SinkArgs& a, const KeyPlan& p, int base, int quad, int ch, bool check,
                                        uint8_t* dst) const {
    bool bad = false;
#pragma unroll
    for (int half = 0; half < C / 8; ++half) {
      const int ch8 = C / 8 * ch + half;
      u32x4 w[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (!kBytes) w[r] = q[r];
        else if constexpr (C == 16) w[r] = kv8_row8(q[r][2 * half], q[r][2 * half + 1], sb[r]);
        else w[r] = kv8_row8(h[r][0], h[r][1], sb[r]);
      }
      if (check) {
        int b0 = base;
        asm volatile("" : "+s"(b0));  // keeps the tests inside this branch
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t keep = key_dead(a, p, b0 + 4 * quad + r) ? 0u : ~0u;
          w[r] &= u32x4{keep, keep, keep, keep};
          bad |= nonfinite2(w[r][0]) || nonfinite2(w[r][1]) || nonfinite2(w[r][2]) || nonfinite2(w[r][3]);
          w[r] = finite_only(w[r]);
        }
      }
      uint8_t* o = dst + (ch8 / 2) * kVTile + (quad % 4) * kVGroup + (ch8 % 2) * 128 + (quad / 4) * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
        *reinterpret_cast<uint2*>(o + 16 * e) = uint2{__builtin_amdgcn_perm(w[1][e / 2], w[0][e / 2], sel),
                                                      __builtin_amdgcn_perm(w[3][e / 2], w[2][e / 2], sel)};
      }
    }
    return bad;
  }
};

__device__ __forceinline__ u32x4 v_operand(const uint8_t* blk, int d, int lane) {
  return *reinterpret_cast<const u32x4*>(blk + d * kVTile + (lane >> 4) * kVGroup + (lane & 15) * 16);
}

// ----------------------------------------------------------------------------- few query rows
// One tile of 16 query rows per workgroup; its split's blocks go round its four waves, each with a running
// state of its own, merged in LDS at the end. No barrier before that: a wave turns its own loads into its
// own operands (4-bit V lies in operand order; row-major V is transposed through the wave's LDS).
// Page ids of 64 blocks are loaded at once, one per lane.
// Bound by the vector units where the cache is quantised: a 32-key block of 128 dims takes a SIMD about 1 us for
// its two waves, most of it the conversion of K and V (two 16-bit values in 4 instructions) and the exponentials;
// bf16 by the loads.

// Waves per SIMD: at head_dim 256 only 4-bit codes fit 256 registers (8 rows of 8192: 66 us with one, 55 with
// two); the others would spill.
template <int HD, int KVT> constexpr int kTileWaves = HD == 128 || KVT == DSK_KV_U4 ? 2 : 1;

// SPREAD, for up to 5 rows: each stands in three columns, which compute the same scores and each take another
// term of the probabilities, so that one product in place of three adds them; the columns are summed at the end
// (us, without / with: 4-bit, one token in 32 rows of 4096, 32 heads 51.4 / 48.1, in 4 rows of 16384 .. 65536
// 56.5 / 54.9, in 8 rows of 8192, 16 heads of 256 50.0 / 47.1; 8-bit, window 4096, 8 rows 24.0 / 23.5).
template <int HD, int KVT, bool SPREAD>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(kTileWaves<HD, KVT>, 2))) void attention_tile_kernel(SinkArgs a) {
  constexpr int KS = HD / 32, DT = HD / 16;
  constexpr int VC = KVT == DSK_KV_U8 ? 16 : 8, NI = HD / VC / 8;  // V items (4 keys x VC dims) per lane
  constexpr bool kRows = KVT != DSK_KV_U4;
  __shared__ __attribute__((aligned(16))) uint8_t lds[kRows && 4 * DT * kVTile > 4 * DT * 1024 ? 4 * DT * kVTile : 4 * DT * 1024];
  __shared__ float2 wml[4][16];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  const int slot = a.by_nkv.quot(blockIdx.x), kvh = blockIdx.x - slot * a.nkv, group = blockIdx.y;
  const SplitTask t = split_task(a, slot, group);
  if (t.live == 0) return;
  const KeyPlan& p = t.p;
  const int r0 = group * a.grows, r = r0 + (SPREAD ? n % kSpreadRows : n), rc = min(r, a.R - 1);
  const float k1 = n >= kSpreadRows ? 1.0f : 0.0f, k2 = n >= 2 * kSpreadRows ? 1.0f : 0.0f;
  const int ri = a.by_G.quot(rc);
  const int pos = p.off + ri, pos_lo = p.off + a.by_G.quot(r0), pos_hi = p.off + a.by_G.quot(min(r0 + 16, a.R) - 1);
  const float c2 = (a.softcap > 0.0f ? 1.0f : a.scale) * kLog2e;
  const Sight see[1] = {sight(a, p, pos)};

  const int nblk = t.v1 > t.v0 + wv ? (t.v1 - t.v0 - wv + 3) / 4 : 0;  // this wave's blocks v0 + wv + 4 i
  uint32_t toks = 0;  // lane l: pool token of block (i & ~63) + l
  auto find_tokens = [&](int i) {
    const int base = p.base(min(t.v0 + wv + 4 * (i + lane), t.v1 - 1));
    const int lp = a.by_page.quot(base), pg = a.block_table[(int64_t)t.b * a.max_pages + lp];
    toks = ((uint32_t)pg * a.nkv + kvh) * a.page + (base - lp * a.page);
  };
  auto token = [&](int i) { return (uint32_t)__builtin_amdgcn_readlane(toks, i & 63); };

  KRaw<HD, KVT> kraw;
  V4Block<HD> v4;
  VRowsRaw<HD, KVT, VC> vr[NI];
  auto quad_of = [](int it) { return (it >> 1) % 8; };  // the bank conflicts of the transposing writes are least so
  auto chunk_of = [](int it) { return (it & 1) + 2 * (it >> 4); };
  auto load_v = [&](uint32_t tok) {
    if constexpr (kRows) {
#pragma unroll
      for (int u = 0; u < NI; ++u) {
        vr[u].load(a, tok, quad_of(lane + 64 * u), chunk_of(lane + 64 * u));
      }
    } else {
      v4.load(a, tok, lane);
    }
  };
  // the queries first: loads return in order, and a wait for them behind K and V would drain those too
  u32x4 qf[KS];
  {
    const uint16_t* src = a.q + ((int64_t)(t.b * a.W + ri) * a.nq + kvh * a.G + rc - ri * a.G) * HD;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = *reinterpret_cast<const u32x4*>(src + KRaw<HD, KVT>::dim(s, g));
  }
  constexpr int kTerms = SPREAD ? 1 : 3;
  Tile<HD, kTerms> tiles[1];
  Tile<HD, kTerms>& tile = tiles[0];
  tile.clear();
  uint8_t* vlds = lds + wv * DT * kVTile;
  if (nblk > 0) {  // the loop within: around it, the count of loads in flight would have to hold for no loads too
    find_tokens(0);
    kraw.load(a, token(0), lane);
    __builtin_amdgcn_sched_barrier(0);
    load_v(token(0));
    int i = 0;
#pragma unroll 1
    do {
      const int base = p.base(t.v0 + wv + 4 * i);
      const bool open = block_open(a, p, base, pos_lo, pos_hi);
      f32x4 st[2] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int x = 0; x < 2; ++x) st[x] = mfma16(kraw.operand(x, s), qf[s], st[x]);
      // the next block (this one again at the end: a load that may not happen would have to be waited for as
      // if it did not)
      const int nx = min(i + 1, nblk - 1);
      const uint32_t tok_now = token(i);
      if (nx > i && (nx & 63) == 0) find_tokens(nx);
      const uint32_t tok_nx = token(nx);
      kraw.load(a, tok_nx, lane);
      if (a.softcap > 0.0f) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) st[x][e] = tanhf(st[x][e] * a.scale / a.softcap) * a.softcap;
      }
      if (!open) mask_scores(see[0], st, 0, base, g);
      const float mx = tile.largest(st, c2);
      if (__any(tile.passes(mx))) tile.raise(mx);
      tile.soften(st[0], st[1], c2);
      u32x4 pt[1][kTerms];
      if constexpr (SPREAD) Tile<HD, kTerms>::own_term(st[0], st[1], k1, k2, pt[0][0]);
      else Tile<HD, kTerms>::terms(st[0], st[1], pt[0]);
      bool bad = false;
      if constexpr (kRows) {
#pragma unroll
        for (int u = 0; u < NI; ++u) {
          vr[u].pin();
          bad |= vr[u].store(a, p, base, quad_of(lane + 64 * u), chunk_of(lane + 64 * u), !open, vlds);
        }
        asm volatile("" ::: "memory");  // a wave's LDS accesses run in order; keep the compiler's order too
      } else {
        v4.pin();
        if (!open) bad = v4.clean(a, p, base, lane);
      }
      if (!open && __any(bad)) add_nonfinite<HD, KVT>(a, tiles, see, pt, base, tok_now, lane);
      static_for<DT / 4>([&](auto q) {
        constexpr int Q = decltype(q)::value, D = 4 * Q;
        u32x4 y[4];
        if constexpr (kRows) {
#pragma unroll
          for (int d = 0; d < 4; ++d) y[d] = v_operand(vlds, D + d, lane);
        } else {
          v4.operands(Q, y);
        }
        tile.template add4<D>(y, pt[0]);
      });
      if constexpr (kRows) asm volatile("" ::: "memory");
      load_v(tok_nx);
    } while (++i < nblk);
  }
  float l = tile.l;
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);

  // ---- the four waves' states merged, each wave a quarter of the d tiles
  __syncthreads();
  f32x4* mo = reinterpret_cast<f32x4*>(lds);  // [wave][d tile][lane]
#pragma unroll
  for (int d = 0; d < DT; ++d) mo[(wv * DT + d) * 64 + lane] = tile.o[d];
  if (g == 0) wml[wv][n] = float2{tile.m, l};
  __syncthreads();
  float M = -__builtin_inff(), L = 0.0f, wq[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) M = fmaxf(M, wml[w][n].x);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    wq[w] = wml[w][n].x == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(wml[w][n].x - M);
    L += wq[w] * wml[w][n].y;
  }
  if (r >= a.R || (SPREAD && n >= kSpreadRows)) return;
  const bool whole = t.live == 1;
  const float inv = L != 0.0f ? 1.0f / L : 0.0f;  // no visible key: zeros; a NaN sum stays NaN
#pragma unroll
  for (int dd = 0; dd < DT / 4; ++dd) {
    const int d = wv * (DT / 4) + dd;
    f32x4 s = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int w = 0; w < 4; ++w)
      if (wq[w] != 0.0f) {
        const f32x4* o = &mo[(w * DT + d) * 64 + lane];
        s += (SPREAD ? o[0] + (o[kSpreadRows] + o[2 * kSpreadRows]) : o[0]) * wq[w];
      }
    if (whole) {
      s *= inv;
      *reinterpret_cast<uint2*>(a.out + sink_out_index(a, HD, t.b, r, kvh, d * 16 + 4 * g)) =
          uint2{pack_bf16x2(s[0], s[1]), pack_bf16x2(s[2], s[3])};
    } else {
      store_part(a.part_o + (((int64_t)t.slot * a.nkv + kvh) * a.R + r) * HD + d * 16 + 4 * g, s);
    }
  }
  if (!whole && wv == 0 && g == 0)
    *reinterpret_cast<float2*>(a.part_ml + (((int64_t)t.slot * a.nkv + kvh) * a.R + r) * 2) = float2{M, L};
}

// ----------------------------------------------------------------------------- many query rows
// NW waves of TPW tiles share each chunk of keys: it is loaded and turned into operands once, into one of
// two LDS buffers, while the other is scored (one barrier per chunk; the chunk after is in flight). Chunks
// are 64 keys at head_dim 128 and 32 at 256, so a buffer is 33 KB: two workgroups of four waves fit a CU.
// Bound by the matrix products (three terms) and the exponentials beside them.
template <int HD> constexpr int kChunkBlocks = HD == 128 ? 2 : 1;

template <int HD, int KVT, int NW, int TPW, int TERMS>
__global__ __launch_bounds__(NW * 64) __attribute__((amdgpu_waves_per_eu(2, 2))) void attention_block_kernel(SinkArgs a) {
  constexpr int KS = HD / 32, DT = HD / 16, NB = kChunkBlocks<HD>, NKT = 2 * NB;
  constexpr bool kRows = KVT != DSK_KV_U4;
  constexpr int kKBytes = NKT * KS * 1024, kVBytes = NB * DT * kVTile;
  __shared__ __attribute__((aligned(16))) uint8_t kbuf[2][kKBytes];
  __shared__ __attribute__((aligned(16))) uint8_t vbuf[2][kVBytes];
  __shared__ int vbad[2][4];  // whether the V unit of a wave held something that is not finite
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 15, g = lane >> 4;
  const int w4 = wv & 3;
  const bool do_k = NW == 4 || wv < 4, do_v = NW == 4 || wv >= 4;
  const int slot = a.by_nkv.quot(blockIdx.x), kvh = blockIdx.x - slot * a.nkv;
  const int group = a.groups - 1 - (int)blockIdx.y;  // the groups with the most keys first
  const SplitTask t = split_task(a, slot, group);
  if (t.live == 0) return;
  const KeyPlan& p = t.p;
  const int r0 = group * a.grows + wv * TPW * 16;
  const bool wave_live = r0 < a.R;
  const int pos_lo = p.off + a.by_G.quot(min(r0, a.R - 1)), pos_hi = p.off + a.by_G.quot(min(r0 + TPW * 16, a.R) - 1);
  // positions of the workgroup's rows: what all of them see is staged as it is
  const int g_lo = p.off + a.by_G.quot(group * a.grows), g_hi = p.off + a.by_G.quot(min(a.R, (group + 1) * a.grows) - 1);
  const float c2 = (a.softcap > 0.0f ? 1.0f : a.scale) * kLog2e;
  const int nch = t.v1 > t.v0 ? (t.v1 - t.v0 + NB - 1) / NB : 0;

  u32x4 qf[TPW][KS];
  Sight see[TPW];
#pragma unroll
  for (int u = 0; u < TPW; ++u) {
    const int rc = min(r0 + 16 * u + n, a.R - 1), ri = a.by_G.quot(rc);
    see[u] = sight(a, p, p.off + ri);
    const uint16_t* src = a.q + ((int64_t)(t.b * a.W + ri) * a.nq + kvh * a.G + rc - ri * a.G) * HD + 8 * g;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[u][s] = *reinterpret_cast<const u32x4*>(src + 32 * s);
  }
  // this thread's pieces of a chunk: K units of (block, tile[, half]) and V units of (block, chunk) for 4-bit
  // codes; 4 K tiles of 16 x 32 and 4 keys x 8 dims of V for rows
  constexpr int kUnits = 4;
  u32x4 kq[kRows ? kUnits : 1];
  uint32_t ksb[kRows ? kUnits : 2];
  V4Raw<HD> v4;
  VRowsRaw<HD, KVT> vr;
  uint32_t tok_next[NB];  // tokens of the chunk to issue next
  auto pool_token = [&](int base) {
    const int lp = a.by_page.quot(base), pg = a.block_table[(int64_t)t.b * a.max_pages + lp];
    return ((uint32_t)pg * a.nkv + kvh) * a.page + (base - lp * a.page);
  };
  auto find = [&](int c) {
#pragma unroll
    for (int u = 0; u < NB; ++u) tok_next[u] = pool_token(p.base(min(t.v0 + c * NB + u, t.v1 - 1)));
  };
  // U4 K unit w4: tile w4 (head_dim 128: of 64 keys), or tile w4 / 2, half w4 % 2 (256); V unit: chunk w4 % (HD / 64) of block w4 / (HD / 64)
  constexpr int kHalves = HD / 128;
  const int kt = w4 / kHalves, kh = w4 % kHalves, vb = w4 / (HD / 64), vc = w4 % (HD / 64);
  const int item = w4 * 64 + lane, vq = (item >> 1) % 8, vch = (item & 1) + 2 * ((item >> 4) % DT), vblk = (item >> 4) / DT;
  auto issue = [&]() {
    if (do_k) {
      if constexpr (kRows) {
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
          const int id = w4 * kUnits + u, kt2 = id / KS, s = id % KS;  // tile, step
          const int64_t row = (int64_t)tok_next[kt2 / 2] + 16 * (kt2 % 2) + n;
          if constexpr (KVT == DSK_KV_BF16) {
            kq[u] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint16_t*>(a.k_pool) + row * HD + 32 * s + 8 * g);
          } else {
            const uint2 x = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(a.k_pool) + row * HD + 32 * s + 8 * g);
            kq[u] = u32x4{x.x, x.y, 0, 0};
            ksb[u] = a.k_sb[row * (HD / 64) + s / 2];
          }
        }
      } else {
        const int64_t row = (int64_t)tok_next[kt / 2] + 16 * (kt % 2) + n;
        kq[0] = *reinterpret_cast<const u32x4*>(reinterpret_cast<const uint8_t*>(a.k_pool) + row * (HD / 2) + 64 * kh + 16 * g);
#pragma unroll
        for (int c = 0; c < 2; ++c) ksb[c] = a.k_sb[row * (HD / 64) + 2 * kh + c];
      }
    }
    if (do_v) {
      if constexpr (kRows) vr.load(a, tok_next[vblk], vq, vch);
      else v4.load(a, tok_next[vb], vc, lane);
    }
  };
  auto stage = [&](int buf, int c) {
    if (do_k) {
      if constexpr (kRows) {
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
          u32x4 w = kq[u];
          if constexpr (KVT == DSK_KV_U8) w = kv8_row8(kq[u][0], kq[u][1], ksb[u]);
          *reinterpret_cast<u32x4*>(&kbuf[buf][(w4 * kUnits + u) * 1024 + lane * 16]) = w;
        }
      } else {
#pragma unroll
        for (int s = 0; s < 4; ++s)
          *reinterpret_cast<u32x4*>(&kbuf[buf][(kt * KS + 4 * kh + s) * 1024 + lane * 16]) = kv4_row8(kq[0][s], kv4_scale(ksb[s / 2]));
      }
    }
    if (do_v) {
      const int blk = kRows ? vblk : vb, v = t.v0 + c * NB + blk;
      const int base = v < t.v1 ? p.base(v) : 0x40000000;  // past the split: every key dead
      const bool check = !block_open(a, p, base, g_lo, g_hi);
      bool bad = false;
      if constexpr (kRows) {
        bad = vr.store(a, p, base, vq, vch, check, &vbuf[buf][blk * DT * kVTile]);
      } else {
        if (check) bad = v4.clean(a, p, base, lane);
        u32x4 x[4];
        v4.operands(x);
#pragma unroll
        for (int d = 0; d < 4; ++d)
          *reinterpret_cast<u32x4*>(&vbuf[buf][(blk * DT + 4 * vc + d) * kVTile + g * kVGroup + n * 16]) = x[d];
      }
      const int any_bad = __any(bad);
      if (lane == 0) vbad[buf][w4] = any_bad;
    }
  };

  Tile<HD, TERMS> tile[TPW];
#pragma unroll
  for (int u = 0; u < TPW; ++u) tile[u].clear();

  auto compute = [&](int buf, int c) {
    int base[NB];
    bool open = true, shut = true;
#pragma unroll
    for (int x = 0; x < NB; ++x) {
      const int v = t.v0 + c * NB + x;
      base[x] = v < t.v1 ? p.base(v) : 0x40000000;
      open &= block_open(a, p, base[x], pos_lo, pos_hi);
      shut &= v >= t.v1 || block_shut(a, base[x], pos_lo, pos_hi);
    }
    if (shut || !wave_live) return;
    f32x4 st[TPW][NKT];
#pragma unroll
    for (int u = 0; u < TPW; ++u)
#pragma unroll
      for (int x = 0; x < NKT; ++x) st[u][x] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int x = 0; x < NKT; ++x) {
        const u32x4 kf = *reinterpret_cast<const u32x4*>(&kbuf[buf][(x * KS + s) * 1024 + lane * 16]);
#pragma unroll
        for (int u = 0; u < TPW; ++u) st[u][x] = mfma16(kf, qf[u][s], st[u][x]);
      }
    float mx[TPW];
    bool up = false;
#pragma unroll
    for (int u = 0; u < TPW; ++u) {
      if (a.softcap > 0.0f) {
#pragma unroll
        for (int x = 0; x < NKT; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) st[u][x][e] = tanhf(st[u][x][e] * a.scale / a.softcap) * a.softcap;
      }
      if (!open) {
#pragma unroll
        for (int x = 0; x < NB; ++x) mask_scores(see[u], st[u], 2 * x, base[x], g);
      }
      mx[u] = tile[u].largest(st[u], c2);
      up |= tile[u].passes(mx[u]);
    }
    if (__any(up)) {
#pragma unroll
      for (int u = 0; u < TPW; ++u) tile[u].raise(mx[u]);
    }
    // a block's exponentials are among the products of the one before
    u32x4 pt[NB][TPW][TERMS];
    auto weigh = [&](auto xc) {
      constexpr int x = decltype(xc)::value;
#pragma unroll
      for (int u = 0; u < TPW; ++u) {
        tile[u].soften(st[u][2 * x], st[u][2 * x + 1], c2);
        Tile<HD, TERMS>::terms(st[u][2 * x], st[u][2 * x + 1], pt[x][u]);
      }
    };
    auto guard = [&](auto xc) {
      constexpr int x = decltype(xc)::value;
      if (open) return;
      bool bad = false;
#pragma unroll
      for (int w = 0; w < 4; ++w) bad |= (kRows ? w * 64 / (16 * DT) : w / (HD / 64)) == x && vbad[buf][w];
      if (bad) add_nonfinite<HD, KVT>(a, tile, see, pt[x], base[x], pool_token(base[x]), lane);
    };
    weigh(std::integral_constant<int, 0>{});
    guard(std::integral_constant<int, 0>{});
    static_for<NB>([&](auto xc) {
      constexpr int x = decltype(xc)::value;
      if constexpr (x + 1 < NB) weigh(std::integral_constant<int, x + 1>{});
      const uint8_t* vb8 = &vbuf[buf][x * DT * kVTile];
      static_for<DT / 4>([&](auto q) {
        constexpr int D = 4 * decltype(q)::value;
        u32x4 w[4];
#pragma unroll
        for (int d = 0; d < 4; ++d) w[d] = v_operand(vb8, D + d, lane);
#pragma unroll
        for (int u = 0; u < TPW; ++u) tile[u].template add4<D>(w, pt[x][u]);
      });
      if constexpr (x + 1 < NB) guard(std::integral_constant<int, x + 1>{});
    });
  };

  if (nch > 0) {
    find(0);
    issue();
    if (nch > 1) find(1);
    stage(0, 0);
    if (nch > 1) issue();
    if (nch > 2) find(2);
    __syncthreads();
    int c = 0;
#pragma unroll 1
    do {
      // half of the waves stage first, so that a SIMD's two waves are not all in products or all out of them
      // (a prompt of 4096 tokens, 32 heads of 128 dims: 289 us with all computing first, 285 so; 2048 tokens
      // under a window of 1024, 12 heads of 256 dims: 107 and 102)
      const bool late = wv >= NW / 2;
      if (!late) compute(c & 1, c);
      if (c + 1 < nch) {
        stage((c + 1) & 1, c + 1);
        if (c + 2 < nch) issue();
        if (c + 3 < nch) find(c + 3);
      }
      if (late) compute(c & 1, c);
      __syncthreads();
    } while (++c < nch);
  }
#pragma unroll
  for (int u = 0; u < TPW; ++u) {
    float l = tile[u].l;
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    const int r = r0 + 16 * u + n;
    if (r >= a.R) continue;
    if (t.live == 1) {
      const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const f32x4 s = tile[u].o[d] * inv;
        *reinterpret_cast<uint2*>(a.out + sink_out_index(a, HD, t.b, r, kvh, d * 16 + 4 * g)) =
            uint2{pack_bf16x2(s[0], s[1]), pack_bf16x2(s[2], s[3])};
      }
    } else {
      const int64_t row = ((int64_t)t.slot * a.nkv + kvh) * a.R + r;
#pragma unroll
      for (int d = 0; d < DT; ++d) store_part(a.part_o + row * HD + d * 16 + 4 * g, tile[u].o[d]);
      if (g == 0) *reinterpret_cast<float2*>(a.part_ml + row * 2) = float2{tile[u].m, l};
    }
  }
}

// ----------------------------------------------------------------------------- splits joined
// One workgroup per (row b, kv head, query row): 256 / (HD / 4) lanes over the splits, 4 dims each, then
// over the lanes in LDS. Splits are added in a fixed order.
// Bound by its chain of loads and the launch: 3.6 us for one row of 16 heads, 4.7 for 4 rows of 16 splits each.
template <int HD>
__global__ __launch_bounds__(256) void attention_join_kernel(SinkArgs a) {
  constexpr int C = HD / 4, S = 256 / C, U = 4;
  __shared__ f32x4 acc_s[S][C];
  __shared__ float2 ml_s[S];
  const int r = blockIdx.x, b = a.by_nkv.quot(blockIdx.y), kvh = blockIdx.y - b * a.nkv;
  const int ch = threadIdx.x % C, sl = threadIdx.x / C;
  int first, live;
  if (a.balanced) {
    const int2 at = a.part_at[b];
    first = at.x;
    live = at.y;
  } else {
    const int group = r / a.grows;
    const int T = key_plan(a, a.seq_lens[b], a.by_G.quot(group * a.grows), a.by_G.quot(min(a.R, (group + 1) * a.grows) - 1)).T;
    const int bps = even_blocks(a, T);
    first = b * a.nsplit;
    live = max(1, (T + bps - 1) / bps);
  }
  if (live == 1) return;  // written whole
  float M = -__builtin_inff(), L = 0.0f;
  f32x4 acc = f32x4{0, 0, 0, 0};
  for (int s0 = sl; s0 < live; s0 += S * U) {
    float2 ml[U];
    f32x4 o[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = min(s0 + u * S, live - 1);
      const int64_t row = ((int64_t)(first + s) * a.nkv + kvh) * a.R + r;
      ml[u] = *reinterpret_cast<const float2*>(a.part_ml + row * 2);
      o[u] = *reinterpret_cast<const f32x4*>(a.part_o + row * HD + ch * 4);
      if (s0 + u * S >= live) ml[u].x = -__builtin_inff();
    }
    float Mn = M;
#pragma unroll
    for (int u = 0; u < U; ++u) Mn = fmaxf(Mn, ml[u].x);
    if (Mn == -__builtin_inff()) continue;
    const float al = M == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(M - Mn);
    L *= al;
    acc *= al;
    M = Mn;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (ml[u].x == -__builtin_inff()) continue;
      const float w = __builtin_amdgcn_exp2f(ml[u].x - M);
      L += w * ml[u].y;
      acc += w * o[u];
    }
  }
  acc_s[sl][ch] = acc;
  if (ch == 0) ml_s[sl] = float2{M, L};
  __syncthreads();
  if (sl > 0) return;
  float Mt = -__builtin_inff(), Lt = 0.0f;
#pragma unroll
  for (int s = 0; s < S; ++s) Mt = fmaxf(Mt, ml_s[s].x);
  f32x4 tot = f32x4{0, 0, 0, 0};
#pragma unroll
  for (int s = 0; s < S; ++s) {
    if (ml_s[s].x == -__builtin_inff()) continue;
    const float w = __builtin_amdgcn_exp2f(ml_s[s].x - Mt);
    Lt += w * ml_s[s].y;
    tot += w * acc_s[s][ch];
  }
  const float inv = Lt != 0.0f ? 1.0f / Lt : 0.0f;
  tot *= inv;
  *reinterpret_cast<uint2*>(a.out + sink_out_index(a, HD, b, r, kvh, ch * 4)) =
      uint2{pack_bf16x2(tot[0], tot[1]), pack_bf16x2(tot[2], tot[3])};
}

// ----------------------------------------------------------------------------- host
// The launch of a pass, from its shape alone (a captured graph replays it for any lengths).
struct SinkPlan {
  bool tile;       // one tile of rows per workgroup, or blocks of rows
  int waves, tpw;  // block kernel
  int groups, grows, nsplit, balanced, slots;
};
static SinkPlan sink_plan(int B, int W, int nq, int nkv, int hd, int causal, int window, int sinks, int max_ctx,
                          int kv_dtype) {
  SinkPlan s = {};
  const int64_t R = (int64_t)W * (nq / nkv);
  // Few rows: a workgroup per 16 rows, each reading the keys again, keeps more of the chip at work than one with
  // idle waves (us, tiles / blocks, contexts of 4096, 32 heads of 128: 8 x 8 new tokens over 4-bit codes 31 / 40,
  // 32 x 8 81 / 131, 32 x 9 118 / 137, 8 x 16 48 / 47; 16 x 8 over 8-bit ones in a window of 4096 59 / 76, 16 x 9
  // 85 / 81; over bf16 91 / 74, at 256 dims in a window of 1024 28 / 34).
  s.tile = R <= (kv_dtype == DSK_KV_U4 ? 64 : kv_dtype == DSK_KV_U8 || hd == 256 ? 32 : 16);
  // keys a pass may look at (the sliding window's rows, and its sinks)
  int64_t span = max_ctx;
  if (causal && window > 0) span = std::min<int64_t>(span, (int64_t)window + W + sinks + 96);
  if (!s.tile) {
    // 256 rows per workgroup share a key's operands, 64 balance better: 256 where they fill the chip unsplit or
    // there are many keys (us, 256 / 64: prompts of 4000 tokens 270 / 341, of 2048 157 / 114, of 1024 82 / 42;
    // 1024 after 16384 543 / 728; verify passes of 17 .. 63 tokens are a tenth slower in 256)
    const bool big = hd == 128 && R >= 256 && ((int64_t)B * nkv * ceil_div(R, 256) > 256 || span >= 4096);
    s.waves = big ? 8 : 4;
    s.tpw = big ? 2 : 1;
  }
  s.grows = s.tile ? 16 : s.waves * s.tpw * 16;
  s.groups = (int)ceil_div(R, s.grows);
  // Splits of many rows are 512 keys or more: their parts are written and read again (200 tokens after 4096:
  // 86 us with at least 1024, 73 so; 512 tokens alone: 39 with at least 256, 22 so).
  const int64_t most = std::max<int64_t>(1, !s.tile && R >= 256 ? span / 512 : ceil_div(ceil_div(span, 32) + 1, kSplitUnit));
  // workgroups that run at once: two per CU; one of 8 waves, or of the tile kernel with one wave per SIMD
  // (2048 tokens after 8192: 620 us planned for two, 586 so)
  const bool one = s.tile ? hd == 256 && kv_dtype != DSK_KV_U4 : s.waves == 8;
  const int64_t tasks = (int64_t)B * nkv * s.groups, want = one ? 256 : 512;
  s.nsplit = (int)std::min<int64_t>(most, std::max<int64_t>(1, want / tasks));
  s.slots = B * s.nsplit;
  if ((s.groups == 1 || s.tile) && B <= kBalancedRows && B > 1) {
    s.slots = (int)std::min<int64_t>(B * most, std::max<int64_t>(B, want / (nkv * s.groups)));
    s.balanced = s.slots > B;
  }
  return s;
}
static size_t sink_part_o_bytes(const SinkPlan& s, int64_t R, int nkv, int hd) {
  return ((size_t)s.slots * nkv * R * hd * sizeof(float) + 255) & ~(size_t)255;
}
static size_t sink_ws(const SinkPlan& s, int B, int64_t R, int nkv, int hd) {
  return s.slots > B ? sink_part_o_bytes(s, R, nkv, hd) + (size_t)s.slots * nkv * R * 2 * sizeof(float) + (s.balanced ? B * sizeof(int2) : 0) : 0;
}

template <int HD, int KVT>
static void launch_sinks(const SinkArgs& a, const SinkPlan& s, int terms, hipStream_t st) {
  const dim3 grid((unsigned)(s.slots * a.nkv), (unsigned)s.groups);
  if (s.tile) {
    constexpr bool kSpread = KVT != DSK_KV_BF16;  // bf16 waits for its loads and gains nothing
    if (kSpread && a.R <= kSpreadRows) hipLaunchKernelGGL((attention_tile_kernel<HD, KVT, kSpread>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((attention_tile_kernel<HD, KVT, false>), grid, dim3(256), 0, st, a);
  } else if (s.waves == 8) {
    if constexpr (HD == 128) {
      if (terms == 2) hipLaunchKernelGGL((attention_block_kernel<HD, KVT, 8, 2, 2>), grid, dim3(512), 0, st, a);
      else hipLaunchKernelGGL((attention_block_kernel<HD, KVT, 8, 2, 3>), grid, dim3(512), 0, st, a);
    }
  } else if (terms == 2) {
    hipLaunchKernelGGL((attention_block_kernel<HD, KVT, 4, 1, 2>), grid, dim3(256), 0, st, a);
  } else {
    hipLaunchKernelGGL((attention_block_kernel<HD, KVT, 4, 1, 3>), grid, dim3(256), 0, st, a);
  }
  if (s.slots > a.B)
    hipLaunchKernelGGL((attention_join_kernel<HD>), dim3((unsigned)a.R, (unsigned)(a.B * a.nkv)), dim3(256), 0, st, a);
}

}  // namespace dsk

using namespace dsk;

extern "C" size_t dsk_attention_sinks_ws_bytes(int B, int W, int nq, int nkv, int hd, int causal, int window, int sinks,
                                               int max_ctx) {
  if (B <= 0 || W <= 0 || nq <= 0 || nkv <= 0 || nq % nkv || (hd != 128 && hd != 256) || max_ctx <= 0 || window < 0 || sinks < 0)
    return 0;
  size_t most = 0;  // of the cache types
  for (int kv : {DSK_KV_BF16, DSK_KV_U8, DSK_KV_U4})
    most = std::max(most, sink_ws(sink_plan(B, W, nq, nkv, hd, causal, window, sinks, max_ctx, kv), B, (int64_t)W * (nq / nkv), nkv, hd));
  return most;
}

extern "C" int dsk_attention_sinks(const uint16_t* q, int B, int W, int nq, int nkv, int hd, float scale, int causal,
                                   int window, int sinks, float softcap, int p_terms, const int32_t* seq_lens,
                                   int max_ctx, const int32_t* block_table, int max_pages, int page, int kv_dtype,
                                   const void* k_pool, const void* v_pool, const uint32_t* k_sb, const uint32_t* v_sb,
                                   uint16_t* out, int out_packed, void* workspace, size_t ws_bytes,
                                   dsk_stream_t stream) {
  const char* who = "dsk_attention_sinks";
  DSK_REQUIRE(q && seq_lens && block_table && k_pool && v_pool && out, "%s: null pointer", who);
  DSK_REQUIRE(hd == 128 || hd == 256, "%s: head_dim %d not supported (128, 256)", who, hd);
  DSK_REQUIRE(B > 0 && W > 0 && nq > 0 && nkv > 0 && nq % nkv == 0, "%s: bad shape", who);
  DSK_REQUIRE(scale > 0.0f && softcap >= 0.0f, "%s: scale must be positive, softcap not negative", who);
  DSK_REQUIRE(p_terms == 3 || (p_terms == 2 && W > kDecodeMaxW), "%s: %d terms of a probability (3; 2 for more than %d new "
              "tokens)", who, p_terms, kDecodeMaxW);
  DSK_REQUIRE(window >= 0 && sinks >= 0 && window < 0x20000000 && sinks < 0x20000000, "%s: window %d, sinks %d", who, window, sinks);
  DSK_REQUIRE(kv_dtype == DSK_KV_BF16 || kv_dtype == DSK_KV_U8 || kv_dtype == DSK_KV_U4, "%s: kv_dtype %d", who, kv_dtype);
  DSK_REQUIRE(kv_dtype == DSK_KV_BF16 || (k_sb && v_sb), "%s: quantised KV needs scale/bias buffers", who);
  DSK_REQUIRE(page > 0 && page % kKv4Block == 0 && max_pages > 0, "%s: pages are multiples of %d tokens (got %d)", who, kKv4Block,
              page);
  DSK_REQUIRE(max_ctx >= W && (int64_t)max_pages * page >= max_ctx && (int64_t)max_pages * page < 0x20000000,
              "%s: max_ctx %d beyond block table", who, max_ctx);
  DSK_REQUIRE((((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)out) & 15) == 0,
              "%s: q, pools and out must be 16-byte aligned", who);
  DSK_REQUIRE(!out_packed || (B * W <= 64 && (nq * hd) % 64 == 0), "%s: packed output needs B*W <= 64", who);
  const int64_t R = (int64_t)W * (nq / nkv);
  const SinkPlan s = sink_plan(B, W, nq, nkv, hd, causal, window, sinks, max_ctx, kv_dtype);
  DSK_REQUIRE(R <= 0x7fffffff && s.groups <= 65535 && (int64_t)s.slots * nkv <= 0x7fffffff && (int64_t)B * nkv <= 65535,
              "%s: %lld query rows per kv head", who, (long long)R);
  const size_t need = sink_ws(s, B, R, nkv, hd);
  if (need && (!workspace || ws_bytes < need)) {
    set_error("%s: workspace %zu < %zu", who, ws_bytes, need);
    return DSK_ENOWS;
  }
  DSK_REQUIRE(((uintptr_t)workspace & 15) == 0 || need == 0, "%s: workspace must be 16-byte aligned", who);
  SinkArgs a = {q, B, W, nq, nkv, nq / nkv, (int)R, scale, softcap, causal ? 1 : 0, window, sinks, seq_lens, block_table,
                max_pages, page, k_pool, v_pool, k_sb, v_sb, out, out_packed ? 1 : 0, s.groups, s.grows, s.slots, s.nsplit,
                s.balanced, reinterpret_cast<float*>(workspace),
                reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + sink_part_o_bytes(s, R, nkv, hd)),
                reinterpret_cast<int2*>(reinterpret_cast<char*>(workspace) + sink_part_o_bytes(s, R, nkv, hd) +
                                        (size_t)s.slots * nkv * R * 2 * sizeof(float)),
                FastDiv(page), FastDiv(nq / nkv), FastDiv(nkv), FastDiv(s.nsplit)};
#define DSK_SINKS(HDV)                                                                                \
  if (kv_dtype == DSK_KV_BF16) launch_sinks<HDV, DSK_KV_BF16>(a, s, p_terms, as_stream(stream));      \
  else if (kv_dtype == DSK_KV_U8) launch_sinks<HDV, DSK_KV_U8>(a, s, p_terms, as_stream(stream));     \
  else launch_sinks<HDV, DSK_KV_U4>(a, s, p_terms, as_stream(stream))
  if (hd == 128) {
    DSK_SINKS(128);
  } else {
    DSK_SINKS(256);
  }
#undef DSK_SINKS
  DSK_LAUNCH_CHECK(who);
  return DSK_OK;
}
