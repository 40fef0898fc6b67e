// kv_selected.hip — attention over selected groups of an INT8 pool, with the groups' attention weight
// (chromofold/kv_select.h, cf_kv_paged_attention_selected_async).
//
// Per (sequence, KV head), over the tokens t of the listed groups, query heads h of the KV head:
//   s_ht = scale q_h . (ks_page (sym - 128)_t),  p = softmax_t(s),  o_h = sum_t p_ht vs_page (sym - 128)_t,
//   weights_out[g] = decay weights_in[g] + sum_h sum_{t in g} p_ht.
// One pass over the blobs with a running maximum and sum per wavefront; wavefronts are joined in LDS, workgroups by a second
// small launch, which also turns the groups' (maximum, sum) pairs into weights.
//
// A wavefront takes one 64-token group (16.4 KB at D = 128) at a time, both products on v_mfma_f32_16x16x32_f16 with the 16
// rows = query heads, so up to 16 of them cost what one does:
//   K  16-byte loads, 1 KiB of the blob each: lane (b, n) = 16 b + n receives quads (4 dims) 4 m + b of the tokens
//      4 n .. 4 n + 3. Word i of two such loads is the lane's 8 k-values of column tile i, whose columns n are the tokens
//      4 n + i; the query operand is laid out to match. The lane ends up with the scores of the tokens 4 n .. 4 n + 3 (one
//      page) for the heads 4 b .. 4 b + 3.
//   V  4-byte loads, 256 B each: lane (G, t) receives tokens 4 q .. 4 q + 3 of page G at dim t + 16 i, i.e. column t of dim
//      tile i and, from two loads, the 8 tokens 8 p .. 8 p + 7 of page G as k-values; the weights go through LDS from the
//      score layout to that of an A operand (16 heads, 8 consecutive tokens a lane).
// Symbols become exact signed f16 (1024 + symbol by v_perm, minus 1152). Queries and weights are f16 hi + lo pairs of
// their fp32 values (22 bits), one MFMA each into the same fp32 accumulator: with single f16 operands the outputs would be
// off by 2^-11, far more than the fp32 they are held in.
// The next group's K is loaded as soon as the current scores are formed, its V after the current P.V: about one whole
// group in flight per wavefront at any time.
#include <algorithm>
#include <cmath>

#include "cf_device.hpp"
#include "chromofold/kv_select.h"

namespace {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));

constexpr int kHdr = 64;
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kRows = 16;
constexpr int kPStride = 80;  // halves of a row of the weight tile: the four rows a store instruction writes start 32 banks apart
constexpr float kLog2e = 1.44269504088896340736f;

struct SelArgs {
  cf_kv_batched_desc d;
  cf_kv_selection s;
  uint32_t slots;    // list entries (groups) of a row: max_units * unit_groups, or max_groups without a list
  uint32_t splits;   // workgroups of a row
  uint32_t per;      // slots of a workgroup
  float *states;     // [row][split][gqa][D + 2]: sum of p v, then maximum (log2 units) and sum of p
  float2 *stats;     // [row][slot][gqa]: a group's maximum (log2 units) and sum of exp2(score - maximum)
};

__device__ __forceinline__ uint32_t visible_tokens(uint32_t tokens, uint32_t pos, uint32_t max_groups) {
  if (tokens == 0) return 0;
  return min(min(tokens - 1, pos), 64 * max_groups - 1) + 1;
}

__device__ __forceinline__ uint32_t as_u32(half2_t h) { return __builtin_bit_cast(uint32_t, h); }
__device__ __forceinline__ half2_t as_half2(uint32_t u) { return __builtin_bit_cast(half2_t, u); }

// Two words of 4 symbols (offset 128) as 8 exact signed f16.
__device__ __forceinline__ half8_t signed_half8(uint32_t w0, uint32_t w1) {
  const half2_t off = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
  uint4_t r;
  r[0] = as_u32(as_half2(__builtin_amdgcn_perm(0x64646464u, w0, 0x04010400u)) + off);
  r[1] = as_u32(as_half2(__builtin_amdgcn_perm(0x64646464u, w0, 0x04030402u)) + off);
  r[2] = as_u32(as_half2(__builtin_amdgcn_perm(0x64646464u, w1, 0x04010400u)) + off);
  r[3] = as_u32(as_half2(__builtin_amdgcn_perm(0x64646464u, w1, 0x04030402u)) + off);
  return __builtin_bit_cast(half8_t, r);
}

// Group of list entry `slot`, or 0xFFFFFFFF where there is none; `bad` if the list does not ascend there.
__device__ __forceinline__ uint32_t listed_group(const SelArgs &a, const uint32_t *list, uint32_t slot, bool &bad) {
  if (!list) return slot;
  const uint32_t u = slot / a.s.unit_groups, j = slot - u * a.s.unit_groups;
  const uint32_t x = list[u];
  if (u > 0) {
    const uint32_t before = list[u - 1];
    bad |= !(x > before || x == CF_KV_NO_UNIT);
  }
  return x >= a.d.max_groups ? 0xFFFFFFFFu : x * a.s.unit_groups + j;
}

template <int D>
__global__ __launch_bounds__(kThreads, 2) void selected_kernel(SelArgs a) {
  constexpr int kSteps = D / 32;   // k-steps of q . k
  constexpr int kTiles = D / 16;   // dim tiles of p . v
  constexpr int kKLoads = D / 16;  // 16-byte loads of a lane: K
  constexpr int kVLoads = D / 4;   // 4-byte loads of a lane: V
  constexpr int kState = kRows * (D + 2);
  __shared__ union {
    struct {
      _Float16 p[kWaves][2][kRows][kPStride];
    };
    float red[kWaves][kState];
    _Float16 q[2][kRows][D];
  } sh;
  __shared__ float s_unit[kRows];  // log2-unit factor of a row's scores, without the page's scale
  __shared__ float s_m[kWaves][kRows];

  const int lane = threadIdx.x & 63, n = lane & 15, b = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t split = blockIdx.x, head = blockIdx.y, seq = blockIdx.z;
  const uint32_t gqa = a.d.query_head_count / a.d.kv_head_count;
  const size_t row = static_cast<size_t>(seq) * a.d.kv_head_count + head;
  const uint32_t visible = visible_tokens(a.d.seq_tokens[seq], a.d.query_pos[seq], a.d.max_groups);
  const uint32_t ngroups = (visible + 63) / 64;
  const uint32_t s0 = min(split * a.per, a.slots);
  const uint32_t *list = a.s.units ? a.s.units + row * a.s.max_units : nullptr;
  const uint32_t s1 = min(list ? a.slots : ngroups, s0 + a.per);
  const uint32_t *grow = a.d.group_offsets + row * a.d.max_groups;

  // ---- queries: each head's in units of a power of two that puts its largest element into [2^14, 2^15)
  for (int h = wave; h < kRows; h += kWaves) {
    constexpr int kN = D / 64;
    const float *q = a.d.queries + (static_cast<size_t>(seq) * a.d.query_head_count + head * gqa + h) * D;
    float x[kN], top = 0.0f;
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      x[j] = static_cast<uint32_t>(h) < gqa ? q[lane + 64 * j] : 0.0f;
      top = fmaxf(top, fabsf(x[j]));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    const int e = top > 0.0f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) - 15 : 0;
#pragma unroll
    for (int j = 0; j < kN; ++j)
      cfd::split_mul_f16(ldexpf(x[j], -e), 1.0f, sh.q[0][h][lane + 64 * j], sh.q[1][h][lane + 64 * j]);
    if (lane == 0) s_unit[h] = ldexpf(a.d.softmax_scale * kLog2e, e);
  }
  __syncthreads();
  half8_t qh[kSteps], ql[kSteps];  // A operands: row n, dims 4 (8 s + b) .. + 3 and 4 (8 s + 4 + b) .. + 3
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
    auto get = [&](int part) {
      const half4_t x = *reinterpret_cast<const half4_t *>(&sh.q[part][n][4 * (8 * s + b)]);
      const half4_t y = *reinterpret_cast<const half4_t *>(&sh.q[part][n][4 * (8 * s + 4 + b)]);
      return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    qh[s] = get(0);
    ql[s] = get(1);
  }
  float unit[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) unit[r] = s_unit[4 * b + r];
  __syncthreads();  // the query area becomes the weight tiles

  float m_run[4], l_run[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) m_run[r] = -INFINITY, l_run[r] = 0.0f;
  int e_run = -(1 << 20);  // acc holds sums in units of 2^e_run
  float4_t acc[kTiles];
#pragma unroll
  for (int i = 0; i < kTiles; ++i) acc[i] = float4_t{0, 0, 0, 0};
  bool bad = false;

  // The wavefront's slots s0 + wave, + kWaves, ...: 64 of them at a time, one a lane, so that no load of the loop below
  // waits for a list entry or an offset.
  for (uint32_t c0 = s0 + wave; c0 < s1; c0 += 64 * kWaves) {
    const uint32_t mine = c0 + lane * kWaves;
    uint32_t g_l = 0xFFFFFFFFu, off_l = 0;
    if (mine < s1) {
      g_l = listed_group(a, list, mine, bad);
      if (g_l < ngroups) off_l = grow[g_l];
    }
    const bool here = g_l < ngroups;
    uint64_t todo = __builtin_amdgcn_ballot_w64(here);
    if (a.s.weights_out && mine < s1 && !here)
      for (uint32_t h = 0; h < gqa; ++h) a.stats[(row * a.slots + mine) * gqa + h] = float2{-INFINITY, 0.0f};
    if (!todo) continue;

    uint4_t kw[kKLoads];
    uint32_t vw[kVLoads];
    float ks, vs;
    uint32_t tc, codec, dim;
    auto blob_of = [&](int i) {  // (readlane returns an int: offsets from 2^31 on must not be sign-extended)
      return a.d.pool + static_cast<size_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(off_l, i))) * 16;
    };
    auto load_k = [&](const uint8_t *p) {
      codec = *reinterpret_cast<const uint32_t *>(p);
      dim = *reinterpret_cast<const uint16_t *>(p + 20);
      tc = reinterpret_cast<const uint16_t *>(p + 12)[n >> 2];
      ks = reinterpret_cast<const float *>(p + 32)[n >> 2];
      vs = reinterpret_cast<const float *>(p + 48)[n >> 2];
#pragma unroll
      for (int i = 0; i < kKLoads; ++i)
        kw[i] = __builtin_nontemporal_load(reinterpret_cast<const uint4_t *>(p + kHdr) + 64 * i + lane);
    };
    auto load_v = [&](const uint8_t *p) {
#pragma unroll
      for (int i = 0; i < kVLoads; ++i)
        vw[i] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t *>(p + kHdr + 64 * D) + 64 * i + lane);
    };
    int cur = __builtin_ctzll(todo);
    todo &= todo - 1;
    const uint8_t *blob = blob_of(cur);
    load_k(blob);
    load_v(blob);
    for (;;) {
      const int next = todo ? __builtin_ctzll(todo) : -1;
      todo &= todo - 1;
      const uint32_t g = __builtin_amdgcn_readlane(g_l, cur);
      const uint8_t *blob_next = next >= 0 ? blob_of(next) : blob;
      // ---- scores of the tokens 4 n + i (one page per lane) for the heads 4 b + r
      float4_t sc[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[i] = float4_t{0, 0, 0, 0};
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const half8_t k = signed_half8(kw[2 * s][i], kw[2 * s + 1][i]);
          sc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ql[s], k, sc[i], 0, 0, 0);
          sc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(qh[s], k, sc[i], 0, 0, 0);
        }
      bad |= codec != CF_KV_CODEC_INT8 || dim != D;
      // tokens of a page are visible from its first on
      const uint32_t page_end = 64 * g + 16 * (n >> 2) + min(tc, 16u);
      const uint32_t first = 64 * g + 4 * n, end = min(page_end, visible);
      const uint32_t nvis = end > first ? min(end - first, 4u) : 0u;
      const bool page_vis = tc > 0 && 64 * g + 16 * (n >> 2) < visible;
      const float ks0 = ks, vs0 = vs;
      if (next >= 0) load_k(blob_next);
      // ---- online softmax
      float mx[4], p[4][4], sum[4];
      bool moved = false;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float f = unit[r] * ks0;
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i][r] = static_cast<uint32_t>(i) < nvis ? sc[i][r] * f : -INFINITY;
        mx[r] = fmaxf(fmaxf(p[0][r], p[1][r]), fmaxf(p[2][r], p[3][r]));
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        mx[r] = cfd::row16_max(mx[r]);
        moved |= mx[r] > m_run[r];
      }
      // units of the P.V sums: the exponent of the group's largest V scale among its visible pages, less 15, so that
      // weights p vs lie in [0, 2^15) and those down to 2^-29 of that are normal f16 numbers. Sums move to a larger unit
      // at once and to a smaller one when 2^8 below (a factor of a power of two; clamped so that it cannot overflow).
      constexpr int kNone = -(1 << 24);
      const int ep = page_vis ? __builtin_amdgcn_frexp_expf(vs0) - 15 : kNone;
      const int eb = max(max(__builtin_amdgcn_readlane(ep, 0), __builtin_amdgcn_readlane(ep, 4)),
                         max(__builtin_amdgcn_readlane(ep, 8), __builtin_amdgcn_readlane(ep, 12)));
      int e_new = e_run;
      if (eb != kNone && (eb > e_run || eb < e_run - 8)) e_new = max(eb, e_run - 60);
      if (__builtin_amdgcn_ballot_w64(moved) || e_new != e_run) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float mn = fmaxf(m_run[r], mx[r]);
          const float al = m_run[r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m_run[r] - mn);
          m_run[r] = mn;
          l_run[r] *= al;
          const float sc2 = ldexpf(al, max(e_run - e_new, -200));  // 0 before the first visible token
#pragma unroll
          for (int i = 0; i < kTiles; ++i) acc[i][r] *= sc2;
        }
        e_run = e_new;
      }
      const float vsn = page_vis ? ldexpf(vs0, -e_run) : 0.0f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float m = m_run[r] == -INFINITY ? 0.0f : m_run[r];
#pragma unroll
        for (int i = 0; i < 4; ++i) p[i][r] = __builtin_amdgcn_exp2f(p[i][r] - m);  // exp2(-inf) = 0
        sum[r] = (p[0][r] + p[1][r]) + (p[2][r] + p[3][r]);
        l_run[r] += sum[r];
      }
      if (a.s.weights_out) {
        const size_t at = (row * a.slots + c0 + static_cast<uint32_t>(cur) * kWaves) * gqa;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float t = cfd::row16_sum(sum[r]);
          if (n == r && static_cast<uint32_t>(4 * b + r) < gqa) a.stats[at + 4 * b + r] = float2{m_run[r], t};
        }
      }
      if (static_cast<uint32_t>(4 * b) < gqa) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          half4_t hi, lo;
          _Float16 h0, l0, h1, l1, h2, l2, h3, l3;
          cfd::split2_mul_f16(p[0][r], p[1][r], vsn, h0, l0, h1, l1);
          cfd::split2_mul_f16(p[2][r], p[3][r], vsn, h2, l2, h3, l3);
          hi = half4_t{h0, h1, h2, h3};
          lo = half4_t{l0, l1, l2, l3};
          *reinterpret_cast<half4_t *>(&sh.p[wave][0][4 * b + r][4 * n]) = hi;
          *reinterpret_cast<half4_t *>(&sh.p[wave][1][4 * b + r][4 * n]) = lo;
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      // ---- P.V: k-values of lane group b = tokens 8 tp .. 8 tp + 7 of page b
#pragma unroll
      for (int tp = 0; tp < 2; ++tp) {
        const half8_t ph = *reinterpret_cast<const half8_t *>(&sh.p[wave][0][n][16 * b + 8 * tp]);
        const half8_t pl = *reinterpret_cast<const half8_t *>(&sh.p[wave][1][n][16 * b + 8 * tp]);
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
          const half8_t v = signed_half8(vw[2 * tp * kTiles + i], vw[(2 * tp + 1) * kTiles + i]);
          acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl, v, acc[i], 0, 0, 0);
          acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, v, acc[i], 0, 0, 0);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      if (next < 0) break;
      load_v(blob_next);
      cur = next;
      blob = blob_next;
    }
  }

  // ---- join the wavefronts
#pragma unroll
  for (int r = 0; r < 4; ++r) l_run[r] = cfd::row16_sum(l_run[r]);
  const bool broken = __builtin_amdgcn_ballot_w64(bad) != 0;
  if (n == 0) {
#pragma unroll
    for (int r = 0; r < 4; ++r)  // a NaN score leaves the maximum as it was and makes the sum a NaN
      s_m[wave][4 * b + r] = broken || l_run[r] != l_run[r] ? __builtin_nanf("") : m_run[r];
  }
  __syncthreads();  // (and the weight tiles are dead)
  if (static_cast<uint32_t>(4 * b) < gqa) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float *o = sh.red[wave] + (4 * b + r) * (D + 2);
#pragma unroll
      for (int i = 0; i < kTiles; ++i) o[16 * i + n] = ldexpf(acc[i][r], max(e_run, -200));
      if (n == 0) o[D] = l_run[r];
    }
  }
  __syncthreads();
  float *st = a.states + (row * a.splits + split) * gqa * (D + 2);
  for (uint32_t i = threadIdx.x; i < gqa * D; i += kThreads) {
    const uint32_t h = i / D, dd = i % D;
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    bool nan = false;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      nan |= s_m[w][h] != s_m[w][h];
      m = fmaxf(m, s_m[w][h]);
    }
    if (m != -INFINITY)
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        if (s_m[w][h] == -INFINITY) continue;
        const float f = __builtin_amdgcn_exp2f(s_m[w][h] - m);
        l += sh.red[w][h * (D + 2) + D] * f;
        o += sh.red[w][h * (D + 2) + dd] * f;
      }
    if (nan) m = __builtin_nanf("");
    if (a.splits == 1 && !a.s.weights_out) {
      a.d.output[(static_cast<size_t>(seq) * a.d.query_head_count + head * gqa + h) * D + dd] =
          nan ? m : m == -INFINITY ? 0.0f : o / l;
    } else {
      st[h * (D + 2) + dd] = o;
      if (dd == 0) {
        st[h * (D + 2) + D] = m;
        st[h * (D + 2) + D + 1] = l;
      }
    }
  }
}

constexpr int kJoinThreads = 256;

// Joins a row's workgroups and turns group statistics into weights: grid (KV heads, sequences).
template <int D>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(SelArgs a) {
  __shared__ float s_m[kRows], s_l[kRows];
  const uint32_t head = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x;
  const uint32_t gqa = a.d.query_head_count / a.d.kv_head_count;
  const size_t row = static_cast<size_t>(seq) * a.d.kv_head_count + head;
  const float *st = a.states + row * a.splits * gqa * (D + 2);
  const size_t stride = static_cast<size_t>(gqa) * (D + 2);
  for (uint32_t i = tid; i < gqa * D; i += kJoinThreads) {
    const uint32_t h = i / D, dd = i % D;
    const float *p = st + h * (D + 2);
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    bool nan = false;
    for (uint32_t s = 0; s < a.splits; ++s) {
      const float x = p[s * stride + D];
      nan |= x != x;
      m = fmaxf(m, x);
    }
    if (m != -INFINITY)
      for (uint32_t s = 0; s < a.splits; ++s) {
        const float x = p[s * stride + D];
        if (x == -INFINITY) continue;
        const float f = __builtin_amdgcn_exp2f(x - m);
        l += p[s * stride + D + 1] * f;
        o += p[s * stride + dd] * f;
      }
    if (nan) m = __builtin_nanf("");
    a.d.output[(static_cast<size_t>(seq) * a.d.query_head_count + head * gqa + h) * D + dd] =
        nan ? m : m == -INFINITY ? 0.0f : o / l;
    if (dd == 0) {
      s_m[h] = m;
      s_l[h] = l;
    }
  }
  if (!a.s.weights_out) return;
  const uint32_t visible = visible_tokens(a.d.seq_tokens[seq], a.d.query_pos[seq], a.d.max_groups);
  const uint32_t ngroups = (visible + 63) / 64;
  const float *in = a.s.weights_in ? a.s.weights_in + row * a.d.max_groups : nullptr;
  float *out = a.s.weights_out + row * a.d.max_groups;
  const uint32_t *list = a.s.units ? a.s.units + row * a.s.max_units : nullptr;
  for (uint32_t g = tid; g < a.d.max_groups; g += kJoinThreads) out[g] = in ? a.s.decay * in[g] : 0.0f;
  __syncthreads();  // s_m, s_l; the decayed weights of the whole row
  for (uint32_t s = tid; s < (list ? a.slots : ngroups); s += kJoinThreads) {
    bool bad = false;
    const uint32_t g = listed_group(a, list, s, bad);
    if (g >= ngroups) continue;
    float w = 0.0f;
    for (uint32_t h = 0; h < gqa; ++h) {
      const float2 x = a.stats[(row * a.slots + s) * gqa + h];
      if (x.x != -INFINITY) w += x.y * __builtin_amdgcn_exp2f(x.x - s_m[h]) / s_l[h];
    }
    out[g] += w;
  }
}

struct Plan {
  uint32_t slots, splits, per;
  uint64_t state_bytes, stat_bytes;
};

Plan make_plan(const cf_kv_batched_desc *d, const cf_kv_selection *s) {
  Plan p{};
  p.slots = d->max_groups;
  if (s->units) p.slots = s->max_units * s->unit_groups;
  const uint64_t rows = static_cast<uint64_t>(d->seq_count) * d->kv_head_count;
  uint32_t splits = d->splits;
  if (splits == 0) {
    // one resident round of wavefronts (two workgroups of four per CU) where there are few slots, at most 16 slots a
    // wavefront where there are many
    const uint64_t per_wave = std::min<uint64_t>(16, std::max<uint64_t>(1, rows * p.slots / (8ull * cfd::cu_count())));
    splits = static_cast<uint32_t>((p.slots + per_wave * kWaves - 1) / (per_wave * kWaves));
  }
  splits = std::max<uint32_t>(1, std::min(splits, p.slots));
  p.per = (p.slots + splits - 1) / splits;
  p.splits = (p.slots + p.per - 1) / p.per;
  const uint32_t gqa = d->query_head_count / d->kv_head_count;
  const bool states = p.splits > 1 || s->weights_out;
  p.state_bytes = states ? (rows * p.splits * gqa * (d->head_dim + 2) * sizeof(float) + 15) / 16 * 16 : 0;
  p.stat_bytes = s->weights_out ? rows * p.slots * gqa * sizeof(float2) : 0;
  return p;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <int D>
void launch(const SelArgs &a, hipStream_t s) {
  selected_kernel<D><<<dim3(a.splits, a.d.kv_head_count, a.d.seq_count), kThreads, 0, s>>>(a);
  if (a.splits > 1 || a.s.weights_out)
    join_kernel<D><<<dim3(a.d.kv_head_count, a.d.seq_count), kJoinThreads, 0, s>>>(a);
}

}  // namespace

extern "C" cf_status cf_kv_validate_selection(const cf_kv_batched_desc *d, const cf_kv_selection *s) {
  if (!s || s->struct_size != sizeof(cf_kv_selection) || s->abi_version != CF_KV_SELECT_ABI_VERSION)
    return CF_ERR_INVALID_ARGUMENT;
  const cf_status v = cf_kv_validate_batched_desc(d);
  if (v != CF_OK) {
    // all that this call takes and the batched one does not: more query heads per KV head, in an INT8 pool
    if (v != CF_ERR_UNSUPPORTED || d->codec != CF_KV_CODEC_INT8 ||
        d->query_head_count / d->kv_head_count > CF_KV_SELECT_MAX_GQA)
      return v;
    cf_kv_batched_desc fewer = *d;
    fewer.query_head_count = d->kv_head_count;
    const cf_status w = cf_kv_validate_batched_desc(&fewer);
    if (w != CF_OK) return w;
  }
  if (d->codec != CF_KV_CODEC_INT8) return CF_ERR_UNSUPPORTED;
  if (d->max_groups == 0) return CF_ERR_INVALID_ARGUMENT;
  if (d->max_groups >= 1u << 26) return CF_ERR_UNSUPPORTED;
  if (s->units) {
    if (s->max_units == 0 || (s->unit_groups != 1 && s->unit_groups != 2)) return CF_ERR_INVALID_ARGUMENT;
    if (s->max_units >= 1u << 26) return CF_ERR_UNSUPPORTED;
  }
  if (!std::isfinite(s->decay) || (s->weights_in && !s->weights_out)) return CF_ERR_INVALID_ARGUMENT;
  return CF_OK;
}

extern "C" uint64_t cf_kv_selected_workspace_bytes(const cf_kv_batched_desc *d, const cf_kv_selection *s) {
  if (cf_kv_validate_selection(d, s) != CF_OK) return 0;
  const Plan p = make_plan(d, s);
  return p.state_bytes + p.stat_bytes;
}

extern "C" cf_status cf_kv_paged_attention_selected_async(const cf_kv_batched_desc *d, const cf_kv_selection *s, void *stream) {
  const cf_status v = cf_kv_validate_selection(d, s);
  if (v != CF_OK) return v;
  const Plan p = make_plan(d, s);
  const uint64_t need = p.state_bytes + p.stat_bytes;
  if (need && (!d->workspace || d->workspace_bytes < need || !aligned16(d->workspace))) return CF_ERR_INVALID_ARGUMENT;
  SelArgs a{*d, *s, p.slots, p.splits, p.per, static_cast<float *>(d->workspace),
            reinterpret_cast<float2 *>(static_cast<char *>(d->workspace) + p.state_bytes)};
  if (!s->units) a.s.unit_groups = 1;
  const hipStream_t st = cfd::as_stream(stream);
  if (d->head_dim == 128) launch<128>(a, st);
  else launch<64>(a, st);
  return cfd::launch_status();
}
