// kv_group_body.hpp — one page group through K scores, softmax and P.V by one wavefront (format 4 and INT8 groups of
// kv_codec_ext.h), shared by the batched decode (kv_batched.hip) and the attention over selected groups of a coded pool
// (kv_selected.hip). What it does and why stands at the head of kv_batched.hip.
#pragma once

#include <hip/hip_fp16.h>

#include <cmath>
#include <utility>

#include "cf_device.hpp"
#include "chromofold/kv_codec_ext.h"
#include "kv_group_decode.hpp"

namespace cfkv {

typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef float float4_t __attribute__((ext_vector_type(4)));

constexpr int kGqa = 4;            // MFMA rows: query heads of one KV head (gqa < 4 pads with zero queries)
constexpr float kOffset = 1152.0f;  // f16 operand = 1024 + symbol, symbol = q + 128

__device__ __forceinline__ half4_t bytes_to_half4(uint32_t b) {
  const uint32_t lo = __builtin_amdgcn_perm(0x64646464u, b, 0x04010400u);  // [s0,0x64,s1,0x64]
  const uint32_t hi = __builtin_amdgcn_perm(0x64646464u, b, 0x04030402u);  // [s2,0x64,s3,0x64]
  half4_t h;
  uint32_t *w = reinterpret_cast<uint32_t *>(&h);
  w[0] = lo;
  w[1] = hi;
  return h;
}

// The same bytes as exact signed values (symbol - 128) in f16: the 1024 + 128 offset removed by a packed f16
// subtract (exact: integers in [-128, 127]). The V operand uses this form: with the offset left in, a row whose
// heaviest tokens have V = 0 would carry 1152 x (sum of their weights) in an fp32 accumulator whose true value
// is many orders of magnitude smaller.
__device__ __forceinline__ half4_t bytes_to_half4_signed(uint32_t b) {
  const half4_t off = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f),
                       static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
  return bytes_to_half4(b) + off;
}

__device__ __forceinline__ float4_t mfma4(half4_t a, half4_t b, float4_t c) {
  return __builtin_amdgcn_mfma_f32_4x4x4f16(a, b, c, 0, 0, 0);
}

// Exact f16 operand of four sign-magnitude values: the f16 denormals (sign << 15) | |q| = q * 2^-24.
__device__ __forceinline__ half4_t sm_to_half4(uint32_t mag, uint32_t signs) {
  half4_t h;
  uint32_t *w = reinterpret_cast<uint32_t *>(&h);
  w[0] = __builtin_amdgcn_perm(signs, mag, 0x05010400u);  // [|q0|, s0, |q1|, s1]
  w[1] = __builtin_amdgcn_perm(signs, mag, 0x07030602u);
  return h;
}

constexpr uint32_t kCapWords = CF_KV_RANS_MAX_GROUP_WORDS;  // K+V words staged in LDS per wavefront
constexpr uint32_t kSlackWords = 64;     // reads past the last word by non-renormalising lanes stay in the buffer

template <int D>
constexpr int raw_words() {  // u32 raw words of one stream of a RANS group
  return raw_words_of(D);
}

template <int D>
constexpr int buf_u32() {
  constexpr int words = (kCapWords + kSlackWords) / 2;
  constexpr int red = kGqa * (D + 2);
  return words > red ? words : red;
}

// Max over the 64 lanes of four values at once, as wave-uniform values: v_max_f32_dpp within each row (quad_perm
// [1,0,3,2], [2,3,0,1], row_half_mirror, row_mirror), then row_bcast:15 (rows 1, 3) and row_bcast:31 (rows 2, 3)
// fold the rows into lane 63, which is read. One asm statement, so that nothing the compiler emits lands between
// the steps: the four chains are interleaved, so each DPP source was written three VALU instructions earlier, and
// the leading s_nop 1 gives the two wait states a DPP read needs after the write of its source before the block.
// Replaces six rounds of ds_bpermute (an LDS round trip each) on the softmax's dependency chain: -2 to -3 % per
// launch at C4.
__device__ __forceinline__ void wave64_max4(float (&x)[4]) {
#define CF_DPP4(CTL)                                                                                                \
  "v_max_f32_dpp %0, %0, %0 " CTL "\n\tv_max_f32_dpp %1, %1, %1 " CTL "\n\tv_max_f32_dpp %2, %2, %2 " CTL        \
  "\n\tv_max_f32_dpp %3, %3, %3 " CTL "\n\t"
  asm volatile("s_nop 1\n\t"
               CF_DPP4("quad_perm:[1,0,3,2] row_mask:0xf bank_mask:0xf")
               CF_DPP4("quad_perm:[2,3,0,1] row_mask:0xf bank_mask:0xf")
               CF_DPP4("row_half_mirror row_mask:0xf bank_mask:0xf")
               CF_DPP4("row_mirror row_mask:0xf bank_mask:0xf")
               CF_DPP4("row_bcast:15 row_mask:0xa bank_mask:0xf")
               CF_DPP4("row_bcast:31 row_mask:0xc bank_mask:0xf")
               : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]));
#undef CF_DPP4
#pragma unroll
  for (int h = 0; h < 4; ++h) x[h] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x[h]), 63));
}

// Units of a wavefront's P.V sums: acc holds them in units of 2^e, and they are below 2^(top + 54); see kDrop. CODED launches
// keep both in one register and settle `top` at the start of a group, others in two and at its end: these kernels' steps
// overlap as far as their registers go, and a register or a branch more elsewhere costs 2-4 % (256 sequences behind a shared
// prefix 156.5 us, 160-163 the other way; INT8 hd 64 17.3, 17.8 the other way).
template <bool CODED>
struct VUnit {
  int e_ = -(1 << 20), top_ = -(1 << 20);
  __device__ __forceinline__ int e() const { return e_; }
  __device__ __forceinline__ int top() const { return top_; }
  __device__ __forceinline__ void set(int e, int top) { e_ = e, top_ = top; }
};
template <>
struct VUnit<true> {
  int both = -(1 << 14) * 65537;
  __device__ __forceinline__ int e() const { return static_cast<int16_t>(both); }
  __device__ __forceinline__ int top() const { return both >> 16; }
  __device__ __forceinline__ void set(int e, int top) { both = (top << 16) | (e & 0xFFFF); }
};

// Decode one page group (K scores, softmax, V accumulation) for `heads` query heads (the other rows hold anything).
// RANS groups: `st` holds the chain's lane states on entry (K, V) and the states the group ends with on return;
// the word streams are read through `wk` (the wave's LDS staging buffer, K stream then V); `raw` points at the
// group's raw words. `pre` holds 14 raw words (7 K + 7 V): on entry the group's first sign group, on return the
// first sign group of the next RANS group at `nlw` (NULL if none); in between, each word of sign group s + 1 is
// loaded into its slot as soon as sign group s no longer needs that slot.
// INT8 groups: `raw` points at the symbol words (offset binary).
// `after_decode` runs as soon as the decode loop no longer needs the word buffer (the caller stages the next group
// there).
// V quads 0..KL-1 do not wait for the V phase in registers: the decode parks them in the wave's LDS area `vl`
// ([KL][64] words) (RANS), or the V phase loads them again from `raw` (INT8 groups, rare in the launches that use
// KL > 0). The registers this frees keep the 12-wave kernel all but free of spills.
// With kEnds (RANS groups), `ends` receives where the K and V word cursors stopped (words from the K stream's start),
// so that a caller can check that a self-contained group consumed exactly its words. With kPageVis, `page_vis`
// tells whether any token of the lane's 16-token page is visible (for callers whose visible tokens are not a prefix
// of each page, e.g. behind a causal window); otherwise tok_ok of the page's first lane says it. kStreamRaw: INT8
// groups' words are read with non-temporal loads (for launches whose groups are each read once). p_out, if given, receives
// the lane's token's weights exp(score - m_run) of the heads. kSelected (the attention over selected groups): pages without
// any visible V do not set the units, which costs the batched decode 3 to 7 %, and groups whose scores are all -inf weigh 0.
template <int D, int CODEC, int KL, typename WordPtr, typename Hook, bool kEnds = false, bool kPageVis = false,
          bool kStreamRaw = false, bool kSelected = false, bool kCoded>
__device__ __forceinline__ void group_body(const Hook &after_decode, uint32_t (&pre)[14], const uint32_t *nlw,
                                           uint32_t (&st)[2], const uint32_t *__restrict__ raw, WordPtr wk,
                                           uint32_t cnt_kv, const uint2 (*__restrict__ s_tab)[kSlots],
                                           const half4_t *qhi, const half4_t *qlo, const float *qsum,
                                           _Float16 (*s_pw)[4][kGqa][16], uint32_t *__restrict__ vl, int lane,
                                           bool tok_ok, float ks, float vs, VUnit<kCoded> &unit, uint32_t heads, float *m_run,
                                           float *l_run, float4_t *acc_v, uint32_t *ends = nullptr, bool page_vis = false,
                                           float *p_out = nullptr) {
  constexpr int NQ = D / 4, RAW = raw_words<D>();
  constexpr bool RANS = CODEC == CF_KV_CODEC_RANS_HYBRID;
  const int G = lane >> 4, t = lane & 15;
  // Where the units of the P.V sums have fallen, the sums as they are say how far they may fall from here: at least by 2^60,
  // unless sums that large are still in them.
  constexpr int kSum = 53, kDrop = 72;
  auto settle = [&] {
    if (unit.top() <= unit.e() + kDrop - 60) return;
    float big = 0.0f;
#pragma unroll
    for (int h = 0; h < kGqa; ++h)
#pragma unroll
      for (int i = 0; i < D / 16; ++i)
        if (static_cast<uint32_t>(h) < heads) big = fmaxf(big, fabsf(acc_v[i][h]));
    big = cfd::rows4_max(cfd::row16_max(big));
    const int e = unit.e(), x = __builtin_amdgcn_readfirstlane(__builtin_amdgcn_frexp_expf(big));
    unit.set(e, big > 0.0f ? max(e, x + e - kSum) : e);
  };
  if constexpr (kCoded) settle();
  float4_t sa = {0, 0, 0, 0}, sb = {0, 0, 0, 0};
  uint32_t vb[NQ];                         // V: magnitude bytes (RANS) or offset-binary symbols (INT8) per quad
  auto put_v = [&](auto qc, uint32_t v) {
    constexpr int q = decltype(qc)::value;
    if constexpr (q < KL) vl[q * 64 + lane] = v;
    else vb[q] = v;
  };
  uint32_t vsg[RANS ? D / 32 : 1];         // V sign words per sign group (RANS)
  // K MFMAs of quad q (A = the 4 query heads broadcast from block q % 16, hi and lo parts)
  auto k_mfma = [&](auto qc, half4_t bk) {
    constexpr int q = decltype(qc)::value;
    sa = __builtin_amdgcn_mfma_f32_4x4x4f16(qhi[q / 16], bk, sa, 4, q % 16, 0);
    sb = __builtin_amdgcn_mfma_f32_4x4x4f16(qlo[q / 16], bk, sb, 4, q % 16, 0);
  };
  if constexpr (RANS) {
    uint32_t xk = st[0], xv = st[1];
    // word cursors of the two streams (wave-uniform: scalar registers; their advance is scalar work)
    const uint32_t ckv = __builtin_amdgcn_readfirstlane(cnt_kv);
    WordPtr wkk = wk, wvv = wk + (ckv & 0xFFFFu);
    // pre[] holds this sign group's raw words (K N0 N1 C0 N2 N3 C1 S, then V the same); each slot is refilled with
    // the next sign group's word right after its last use here (at least three steps before that word is needed),
    // and the next sign words go to snx at the sign group's first step.
    uint32_t snx[2] = {0, 0};
    auto refill = [&](auto sgc, auto wc) {  // slots w (K) and 7 + w (V) <- word w of sign group sgc + 1
      constexpr int sn = decltype(sgc)::value + 1, w = decltype(wc)::value;
      if constexpr (sn < D / 32) {
        pre[w] = raw[(7 * sn + w) * 64 + lane];
        pre[7 + w] = raw[RAW + (7 * sn + w) * 64 + lane];
      } else if (nlw) {
        pre[w] = nlw[w * 64 + lane];
        pre[7 + w] = nlw[RAW + w * 64 + lane];
      }
    };
    // step P decodes quads 2P and 2P + 1 of K and of V: two independent rANS steps
    [&]<int... P>(std::integer_sequence<int, P...>) {
      (
          [&] {
            constexpr int sg = P / 4, m = P % 4, q0 = 2 * P;
            constexpr uint32_t rA = kFrame[2 * m], rB = kFrame[2 * m + 1];
            using SG = std::integral_constant<int, sg>;
            if constexpr (m == 0) {
              vsg[sg] = pre[13];  // V signs, kept for the V phase
              if constexpr (sg + 1 < D / 32) {
                snx[0] = raw[(7 * (sg + 1) + 6) * 64 + lane];
                snx[1] = raw[RAW + (7 * (sg + 1) + 6) * 64 + lane];
              } else if (nlw) {
                snx[0] = nlw[6 * 64 + lane];
                snx[1] = nlw[RAW + 6 * 64 + lane];
              }
            }
            const uint2 ek = rans_lookup(s_tab[0], xk), ev = rans_lookup(s_tab[1], xv);
            uint32_t selk, selv;
            const uint32_t wdk = rans_advance(ek.x, xk, wkk, selk);
            const uint32_t wdv = rans_advance(ev.x, xv, wvv, selv);
            xk = __builtin_amdgcn_perm(xk, wdk, selk);
            xv = __builtin_amdgcn_perm(xv, wdv, selv);
            // the spread words hold the big bits in the frames (0, 4): rotate them into this pair's frames
            const uint32_t spk = rA ? __builtin_amdgcn_alignbit(ek.y, ek.y, 32 - rA) : ek.y;
            const uint32_t spv = rA ? __builtin_amdgcn_alignbit(ev.y, ev.y, 32 - rA) : ev.y;
            constexpr int nw = kNWord[m], cwi = m < 2 ? 2 : 5;
            k_mfma(std::integral_constant<int, q0>{},
                   sm_to_half4(quad_mag<rA>(pre[nw], pre[cwi], spk), quad_signs<rA>(pre[6])));
            k_mfma(std::integral_constant<int, q0 + 1>{},
                   sm_to_half4(quad_mag<rB>(pre[nw], pre[cwi], spk), quad_signs<rB>(pre[6])));
            put_v(std::integral_constant<int, q0>{}, quad_mag<rA>(pre[7 + nw], pre[7 + cwi], spv));
            put_v(std::integral_constant<int, q0 + 1>{}, quad_mag<rB>(pre[7 + nw], pre[7 + cwi], spv));
            // refill what this step used for the last time in this sign group
            refill(SG{}, std::integral_constant<int, nw>{});
            if constexpr (m == 1 || m == 3) refill(SG{}, std::integral_constant<int, cwi>{});
            if constexpr (m == 3) {
              pre[6] = snx[0];
              pre[13] = snx[1];
            }
          }(),
          ...);
    }(std::make_integer_sequence<int, D / 8>{});
    st[0] = xk;
    st[1] = xv;
    if constexpr (kEnds) {
      ends[0] = static_cast<uint32_t>(wkk - wk);
      ends[1] = static_cast<uint32_t>(wvv - wk);
    }
  } else {
    if (nlw) {  // a raw group: start the next RANS group's first raw words now
#pragma unroll
      for (int w = 0; w < 7; ++w) {
        pre[w] = nlw[w * 64 + lane];
        pre[7 + w] = nlw[RAW + w * 64 + lane];
      }
    }
    // with kStreamRaw the words go past the caches (non-temporal): ~12 % faster at C4's 2.2 GB of INT8 groups read
    // once each, but raw groups that many sequences share (a prefix inside a RANS pool) need the caches
    auto ld = [&](const uint32_t *p) { return kStreamRaw ? __builtin_nontemporal_load(p) : *p; };
    [&]<int... Q>(std::integer_sequence<int, Q...>) {
      ((Q < KL ? void() : void(vb[Q] = ld(&raw[NQ * 64 + Q * 64 + lane])),
        k_mfma(std::integral_constant<int, Q>{}, bytes_to_half4(ld(&raw[Q * 64 + lane])))),
       ...);
    }(std::make_integer_sequence<int, NQ>{});
  }
  after_decode();  // the word buffer is free from here on

  // ---- online softmax over the wavefront's 64 tokens (one running max per head for all four pages)
  // K operands: RANS = q * 2^-24 (f16 denormals); INT8 = 1024 + symbol, the 1152 offset folded out with the query sum
  const float ksc = RANS ? ks * 16777216.0f : ks;
  float s[kGqa], mx[kGqa];
#pragma unroll
  for (int h = 0; h < kGqa; ++h) {
    s[h] = tok_ok ? (RANS ? (sa[h] + sb[h]) : (sa[h] + sb[h] - kOffset * qsum[h])) * ksc : -INFINITY;
    mx[h] = s[h];
  }
  static_assert(kGqa == 4, "wave64_max4 reduces four heads");
  wave64_max4(mx);
  // P.V runs on v_mfma_f32_16x16x32_f16 with k = 8 tokens of each of the 4 pages (page G's from lane group G), so
  // one MFMA sums all four pages: rows 0-3 are the 4 heads' hi parts of the weights p * v_scale, rows 4-7 their lo
  // parts (rows 8-15 repeat rows 0-7 and are dropped), 16 dims per MFMA. The lane's accumulators acc_v hold rows
  // 4G..4G+3: the hi (G = 0) or lo (G = 1) sums. The wavefront keeps them in units of 2^e with e = (exponent of
  // the group's largest V scale among its pages with a visible token) - 15 (+ 24 for RANS groups, whose V operands
  // are q * 2^-24): every f16 weight lies in [0, 2^15) whatever the V magnitude, weights down to 2^-29 of the
  // running maximum stay normal f16 numbers (a row whose heaviest tokens have V = 0 is carried by such small
  // weights), and hi + lo keep ~22 bits for every page within 2^18 of the group's largest V scale (the lo part of a
  // page further below loses bits gradually: ~16 bits at 2^24, those of one f16 at 2^29). Moving to new units is an
  // exact power-of-two factor folded into the softmax rescale. 2^31 tokens of weights below 2^15 and values up to 2^7
  // add up to less than 2^53 of the largest unit so far (unit.top()): in a unit down to 2^-kDrop of it they stay finite.
  constexpr int kOpExp = RANS ? 24 : 0;
  constexpr int kNone = -(1 << 24);
  // tokens are visible as a prefix of each page, so a page's lane 16 G is visible iff any of its tokens is
  int ep = kNone;
  if ((kPageVis ? page_vis : tok_ok) && (!kSelected || vs != 0.0f)) ep = __builtin_amdgcn_frexp_expf(vs) - 15 + kOpExp;
  int eb = max(max(__builtin_amdgcn_readlane(ep, 0), __builtin_amdgcn_readlane(ep, 16)),
               max(__builtin_amdgcn_readlane(ep, 32), __builtin_amdgcn_readlane(ep, 48)));
  // kSelected: where scales lie far apart, pages whose visible V are all 0 (their scale is 1, or anything) are left out, lest
  // the others' weights lose their bits to units that nothing needs.
  if constexpr (kSelected) {
    static_assert(KL == 0, "all V quads in registers");
    if (__builtin_amdgcn_ballot_w64(ep < eb - 8 && ep != kNone)) [[unlikely]] {
      const uint32_t seen = static_cast<uint32_t>(__builtin_amdgcn_ballot_w64(tok_ok) >> (16 * G)) & 0xFFFFu;  // of page G
      uint32_t any = 0;
#pragma unroll
      for (int tq = 0; tq < 4; ++tq) {
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const int q = tq * (D / 16) + i;
          word |= RANS ? vb[q] : vb[q] ^ 0x80808080u;
        }
        any |= word & ((seen >> (4 * tq) & 15u) * 0x00204081u & 0x01010101u) * 255u;
      }
      const uint64_t live = __builtin_amdgcn_ballot_w64(any != 0);
      if ((live >> (16 * G) & 0xFFFFu) == 0 && fabsf(vs) < INFINITY) vs = 0.0f, ep = kNone;
      eb = max(max(__builtin_amdgcn_readlane(ep, 0), __builtin_amdgcn_readlane(ep, 16)),
               max(__builtin_amdgcn_readlane(ep, 32), __builtin_amdgcn_readlane(ep, 48)));
    }
  }
  const int nb = eb != kNone ? max(eb, unit.top() - kDrop) : unit.e();
  const int de = unit.e() - nb;
  unit.set(nb, max(unit.top(), nb));
  // 0 for a token that is not visible: its page's scale may be anything (that of an absent page is 1, which small units
  // make infinite), and 0 * inf would be in every row's sum
  const float vsn = tok_ok ? ldexpf(vs, kOpExp - nb) : 0.0f;
  float alpha[kGqa], pr[kGqa];
#pragma unroll
  for (int h = 0; h < kGqa; ++h) {
    const float mn = fmaxf(m_run[h], mx[h]);
    const float a = (m_run[h] == -INFINITY) ? 0.0f : __expf(m_run[h] - mn);
    // kSelected: 0 as long as every score was -inf, where s - mn would be a NaN
    pr[h] = tok_ok ? __expf(s[h] - (kSelected && mn == -INFINITY ? 0.0f : mn)) : 0.0f;
    l_run[h] = l_run[h] * a + pr[h];
    alpha[h] = ldexpf(a, de);  // ldexp(0, .) = 0 before the first visible token
    m_run[h] = mn;
    if (p_out) p_out[h] = pr[h];
  }
#pragma unroll
  for (int h = 0; h < kGqa; h += 2)
    cfd::split2_mul_f16(pr[h], pr[h + 1], vsn, s_pw[0][G][h][t], s_pw[1][G][h][t], s_pw[0][G][h + 1][t],
                        s_pw[1][G][h + 1][t]);
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
#pragma unroll
    for (int h = 0; h < kGqa; ++h) acc_v[i][h] *= alpha[h];
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");

  // ---- V MFMAs: rows {hi, lo} x heads, k = tokens 8 tp .. 8 tp + 7 of every page, cols = dims 16 i .. 16 i + 15.
  // A: lane (G, t) gives row t for page G (rows 8-15 read rows 0-7's weights); B: its V quads of tokens
  // 8 tp .. + 3 and 8 tp + 4 .. + 7 at dim 16 i + t.
  auto v_quad = [&](auto qc) {
    constexpr int q = decltype(qc)::value;  // quad q = tokens 4 (q / (D / 16)) .. + 3 at dim t + 16 (q % (D / 16))
    if constexpr (RANS)  // quad q is quad q % 8 of sign group q / 8
      return sm_to_half4(q < KL ? vl[q * 64 + lane] : vb[q], quad_signs<kFrame[q % 8]>(vsg[q / 8]));
    else
      return bytes_to_half4_signed(q < KL ? raw[NQ * 64 + q * 64 + lane] : vb[q]);
  };
  [&]<int... TP>(std::integer_sequence<int, TP...>) {
    (
        [&] {
          constexpr int tp = TP;
          // Read in inline asm: the compiler cannot tell this tile from the word buffer that the next group's
          // global_load_lds copies are filling, and for a plain LDS read it would first wait for those copies
          // (s_waitcnt vmcnt(0)), i.e. for the next group's whole prefetch, in the middle of every group. The
          // tile was written by this wavefront's own ds_write instructions, which the LDS executes in order.
          half8_t pa;
          asm volatile("ds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)"
                       : "=v"(pa)
                       : "v"(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(&s_pw[(t >> 2) & 1][G][t & 3][8 * tp])))
                       : "memory");
          [&]<int... I>(std::integer_sequence<int, I...>) {
            (
                [&] {
                  constexpr int i = I;
                  const half4_t b0 = v_quad(std::integral_constant<int, (2 * tp) * (D / 16) + i>{});
                  const half4_t b1 = v_quad(std::integral_constant<int, (2 * tp + 1) * (D / 16) + i>{});
                  const half8_t bv = __builtin_shufflevector(b0, b1, 0, 1, 2, 3, 4, 5, 6, 7);
                  acc_v[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pa, bv, acc_v[i], 0, 0, 0);
                }(),
                ...);
          }(std::make_integer_sequence<int, D / 16>{});
        }(),
        ...);
  }(std::make_integer_sequence<int, 2>{});
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  if constexpr (!kCoded) settle();
}

}  // namespace cfkv
