// kv_selected.hip — attention over selected groups of a pool, with the groups' attention weight
// (chromofold/kv_select.h, cf_kv_paged_attention_selected_async).
//
// The kernels for INT8 pools; the one for RANS_HYBRID pools stands at the end and shares the cuts, joins and weights.
// Per (sequence, KV head), over the tokens t of the listed groups, query heads h of the KV head:
//   s_ht = scale q_h . (ks_page (sym - 128)_t),  p = softmax_t(s),  o_h = sum_t p_ht vs_page (sym - 128)_t,
//   weights_out[g] = decay weights_in[g] + sum_h sum_{t in g} p_ht.
// One pass over the blobs with a running maximum and sum per wavefront; a row's states are joined in LDS or by a second small
// launch, which also turns the groups' (maximum, sum) pairs into weights. Bound by reading the blobs: 32 x 512 groups of all
// 8 heads (2.16 GB) at 6.4 TB/s with that launch, 6.7 as one workgroup per row; with 16 query heads per KV head, whose softmax
// fills all lanes, at 5.5.
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
#include "kv_group_body.hpp"
#include "kv_topk.hpp"

namespace {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float float4_t __attribute__((ext_vector_type(4)));
typedef float float4a4_t __attribute__((ext_vector_type(4), aligned(4)));  // queries need no more than a float's alignment
typedef uint32_t uint4_t __attribute__((ext_vector_type(4)));

constexpr int kHdr = 64;
constexpr int kWaves = 4;     // of a workgroup
constexpr int kWavesRow = 8;  // of a workgroup that takes a whole row
constexpr uint32_t kResident = 8;  // wavefronts of a CU at these kernels' registers
constexpr int kRows = 16;
constexpr int kPStride = 80;  // halves of a row of the weight tile: the four rows a store instruction writes start 32 banks apart
constexpr uint32_t kRowStats = 2048;  // group statistics that a workgroup with a whole row holds in LDS
constexpr uint32_t kSpanSeqs = 1024;  // sequences of a span launch (their prefix sums are made by each workgroup)
constexpr float kLog2e = 1.44269504088896340736f;

// How a launch cuts the rows ((sequence, KV head) pairs, each of some slots: list entries, or groups without a list):
//   kSpan   all rows' slots laid end to end, heads outermost, an equal stretch for each wavefront. The lengths are device
//           memory: a grid over rows is sized for the longest sequence and waits for it, a stretch is equal whatever they are,
//           and a wavefront's loads run on from one row into the next.
//   kRow    a workgroup per row, which finishes it: no second launch
//   kSplit  `splits` workgroups per row, `per` slots each: a row's result depends on its own sequence alone
//   kCoded  kSplit for RANS_HYBRID pools, `per` a multiple of the groups of a unit
enum Mode { kSpan, kRow, kSplit, kCoded };

struct SelArgs {
  cf_kv_batched_desc d;
  cf_kv_selection s;
  uint32_t slots;    // the most slots of a row: max_units * unit_groups list entries, or max_groups without a list
  uint32_t splits;   // kSplit: workgroups of a row
  uint32_t per;      // kSplit: slots of a workgroup
  uint32_t nwaves;   // kSpan: wavefronts
  uint32_t *pre;     // kSpan: [seq_count + 1] prefix sums of the sequences' slots, for the second launch
  float *sums;       // [state][gqa][D]: sum of p v
  float2 *states;    // [state][gqa]: maximum (log2 units) and sum of p
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

// Slots of a row: with a list, the entries that can name a visible unit.
__device__ __forceinline__ uint32_t row_slots(const SelArgs &a, uint32_t ngroups) {
  return a.s.units ? min(a.slots, (ngroups + a.s.unit_groups - 1) / a.s.unit_groups * a.s.unit_groups) : ngroups;
}

// Weight of an attended group from its heads' statistics, the row's maxima and the inverse sums (0 of a group whose scores are
// all -inf; a row of such groups has a NaN for its maximum).
template <typename Stat>
__device__ __forceinline__ float group_weight(const Stat &stat, uint32_t gqa, const float *m, const float *inv_l) {
  float w = 0.0f;
  for (uint32_t h0 = 0; h0 < gqa; h0 += 4) {
    float2 x[4];
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j) x[j] = stat(min(h0 + j, gqa - 1));
#pragma unroll
    for (uint32_t j = 0; j < 4; ++j)
      if (h0 + j < gqa) w += x[j].y * __builtin_amdgcn_exp2f(x[j].x - m[h0 + j]) * inv_l[h0 + j];
  }
  return w;
}

// The row's weights of groups [lo, hi): decayed, then the listed ones' shares added. All threads of the workgroup call this.
template <typename Stat>
__device__ __forceinline__ void write_weights(const SelArgs &a, size_t row, const uint32_t *list, uint32_t ngroups,
                                              uint32_t nslots, uint32_t lo, uint32_t hi, uint32_t gqa, const float *m,
                                              const float *inv_l, const Stat &stat) {
  const float *in = a.s.weights_in ? a.s.weights_in + row * a.d.max_groups : nullptr;
  float *out = a.s.weights_out + row * a.d.max_groups;
  if (!list) {
    for (uint32_t g = lo + threadIdx.x; g < hi; g += blockDim.x) {
      const float w = in ? a.s.decay * in[g] : 0.0f;
      out[g] = g < ngroups ? w + group_weight([&](uint32_t h) { return stat(g, h); }, gqa, m, inv_l) : w;
    }
    return;
  }
  for (uint32_t g = lo + threadIdx.x; g < hi; g += blockDim.x) out[g] = in ? a.s.decay * in[g] : 0.0f;
  __syncthreads();
  for (uint32_t s = threadIdx.x; s < nslots; s += blockDim.x) {
    bool bad = false;
    const uint32_t g = listed_group(a, list, s, bad);
    if (g < ngroups && g >= lo && g < hi) out[g] += group_weight([&](uint32_t h) { return stat(s, h); }, gqa, m, inv_l);
  }
}

// One group's blob on its way: K quads, V quads and the header's fields of this lane's page. The loads are non-temporal: a
// blob is read once (32 x 512 groups 340 against 391 us).
template <int D>
struct Blob {
  uint4_t kw[D / 16];
  uint32_t vw[D / 4];
  float ks, vs;
  uint32_t tc, codec, dim;
  __device__ __forceinline__ void load_k(const uint8_t *p) {
    const int lane = threadIdx.x & 63, n = lane & 15;
    codec = *reinterpret_cast<const uint32_t *>(p);
    dim = *reinterpret_cast<const uint16_t *>(p + 20);
    tc = reinterpret_cast<const uint16_t *>(p + 12)[n >> 2];
    ks = reinterpret_cast<const float *>(p + 32)[n >> 2];
    vs = reinterpret_cast<const float *>(p + 48)[n >> 2];
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
      kw[i] = __builtin_nontemporal_load(reinterpret_cast<const uint4_t *>(p + kHdr) + 64 * i + lane);
  }
  __device__ __forceinline__ void load_v(const uint8_t *p) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < D / 4; ++i)
      vw[i] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t *>(p + kHdr + 64 * D) + 64 * i + lane);
  }
};

// A wavefront's LDS: the weight tile, and statistics of the groups looked up together, on their way to memory in whole
// lines (one group's are 8 bytes a head; written on their own they cost 256 rows of 512 groups 15 of 350 us).
constexpr uint32_t kLookStats = 256;
struct WaveLds {
  _Float16 p[2][kRows][kPStride];
  float2 stat[kLookStats];
};
__device__ __forceinline__ uint32_t look_slots(uint32_t gqa) { return min(64u, kLookStats / gqa); }

// Queries of one row as they lie in memory, in the layout of the A operands: row n, dims 4 (8 s + b) .. + 3 and
// 4 (8 s + 4 + b) .. + 3 of step s.
template <int D>
struct Query {
  float4_t x[D / 16];
  __device__ __forceinline__ void load(const SelArgs &a, uint32_t seq, uint32_t head, uint32_t gqa) {
    const int lane = threadIdx.x & 63, n = lane & 15, b = lane >> 4;
    const float *q = a.d.queries +
                     (static_cast<size_t>(seq) * a.d.query_head_count + head * gqa + min(static_cast<uint32_t>(n), gqa - 1)) * D;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) x[s] = *reinterpret_cast<const float4a4_t *>(q + 4 * (4 * s + b));
  }
};

// How the softmax's work lies in the lanes. The scores come from the MFMAs with the heads 4 b + r in lane group b, a tile of
// 16 tokens per accumulator: with at most 4 heads only one group of lanes has any, 16 of them each. GT = lane groups that the
// heads fill (1, 2 or 4): with fewer than 4 the tiles are dealt out over the idle groups by row exchanges, and a lane
// (b, n) keeps GT scores of each of the heads 4 (b % GT) + r, at the tokens token(j), j < GT. At 4 heads that takes the
// vector instructions of a group from 465 to 366 at D = 64 and from 635 to 537 at D = 128 (32 x 512 groups of hd 64, 1.1 GB:
// 217 -> 189 us).
template <int GT>
struct Spread {
  // exchange of rows: {a0 b0 a2 b2, a1 b1 a3 b3} and {a0 a1 b0 b1, a2 a3 b2 b3}
  static __device__ __forceinline__ void swap16(float &a, float &b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    a = __uint_as_float(r[0]);
    b = __uint_as_float(r[1]);
  }
  static __device__ __forceinline__ void swap32(float &a, float &b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    a = __uint_as_float(r[0]);
    b = __uint_as_float(r[1]);
  }
  static __device__ __forceinline__ uint32_t head(int b, int r) { return 4 * (b % GT) + r; }
  static __device__ __forceinline__ int token(int n, int b, int j) { return 4 * n + (GT == 4 ? j : GT == 2 ? 2 * (b / 2) + j : b); }
  // sc[i][r]: tile i, head 4 b + r -> s[j][r]
  static __device__ __forceinline__ void deal(const float4_t (&sc)[4], float (&s)[GT][4]) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float x[4] = {sc[0][r], sc[1][r], sc[2][r], sc[3][r]};
      if constexpr (GT < 4) {
        swap32(x[0], x[2]);
        swap32(x[1], x[3]);
      }
      if constexpr (GT == 1) swap16(x[0], x[1]);
#pragma unroll
      for (int j = 0; j < GT; ++j) s[j][r] = x[j];
    }
  }
  // Reduces x[r] over all lanes that hold the head of (b, r); every such lane gets the result.
  template <typename Op, typename Row>
  static __device__ __forceinline__ void reduce(float (&x)[4], const Op &op, const Row &row16) {
    if constexpr (GT == 4) {
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = row16(x[r]);
    } else {
      swap32(x[0], x[1]);
      swap32(x[2], x[3]);
      float a = op(x[0], x[1]), c = op(x[2], x[3]);  // halves: heads of r = 0 | 1, and of r = 2 | 3
      if constexpr (GT == 2) {
        a = row16(a);
        c = row16(c);
        x[0] = x[1] = a;
        x[2] = x[3] = c;
        swap32(x[0], x[1]);
        swap32(x[2], x[3]);
      } else {
        swap16(a, c);
        a = row16(op(a, c));  // rows: r = 0, 2, 1, 3
        x[0] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(a), 0));
        x[1] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(a), 32));
        x[2] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(a), 16));
        x[3] = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(a), 48));
      }
    }
  }
  // (fmaxf and not cfd::vmax_f32: a row exchange must not follow within two wait states of the write of what it exchanges,
  // which the compiler sees to for its own instructions only)
  static __device__ __forceinline__ void reduce_max(float (&x)[4]) {
    reduce(x, [](float a, float b) { return fmaxf(a, b); }, [](float a) { return cfd::row16_max(a); });
  }
  static __device__ __forceinline__ void reduce_sum(float (&x)[4]) {
    reduce(x, [](float a, float b) { return a + b; }, [](float a) { return cfd::row16_sum(a); });
  }
};

// A wavefront's running state of one row: maximum and sum of the heads Spread::head(b, r), sums of p v of the heads 4 b + r
// (row r of the accumulators) at dim 16 i + n.
template <int D, int GT>
struct RowState {
  float m[4], l[4];
  int e;    // acc holds sums in units of 2^e
  int top;  // and they are below 2^(top + 54); see kDrop
  float4_t acc[D / 16];
  float unit[4];  // log2-unit factor of the heads' scores, without the page's scale
  half8_t qh[D / 32], ql[D / 32];
  bool bad;

  __device__ __forceinline__ void reset() {
#pragma unroll
    for (int r = 0; r < 4; ++r) m[r] = -INFINITY, l[r] = 0.0f;
    e = top = -(1 << 20);
#pragma unroll
    for (int i = 0; i < D / 16; ++i) acc[i] = float4_t{0, 0, 0, 0};
    bad = false;
  }

  // Each head in units of a power of two that puts its largest element into [2^14, 2^15), as f16 hi + lo.
  __device__ __forceinline__ void set_query(const SelArgs &a, const Query<D> &q, uint32_t gqa) {
    const int lane = threadIdx.x & 63, n = lane & 15, b = lane >> 4;
    float top = 0.0f;
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j) top = fmaxf(top, fabsf(q.x[s][j]));
    top = cfd::rows4_max(top);
    const int x = top > 0.0f && top < INFINITY ? __builtin_amdgcn_frexp_expf(top) - 15 : 0;
    const float u = ldexpf(a.d.softmax_scale * kLog2e, x);
#pragma unroll
    for (int r = 0; r < 4; ++r) unit[r] = __shfl(u, static_cast<int>(Spread<GT>::head(b, r)));
#pragma unroll
    for (int s = 0; s < D / 32; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float v = static_cast<uint32_t>(n) < gqa ? ldexpf(q.x[2 * s + j / 4][j % 4], -x) : 0.0f;
        _Float16 hi, lo;
        cfd::split_mul_f16(v, 1.0f, hi, lo);
        qh[s][j] = hi;
        ql[s][j] = lo;
      }
  }

  // Group g (its K and V in w). next: the blob to load after it, or null. put(h, m, l) receives its statistics if `stats`.
  template <typename Put>
  __device__ __forceinline__ void attend(Blob<D> &w, uint32_t g, uint32_t visible, uint32_t gqa, WaveLds &lds,
                                         const uint8_t *next, bool stats, const Put &put) {
    constexpr int kTiles = D / 16;
    const int lane = threadIdx.x & 63, n = lane & 15, b = lane >> 4;
    // ---- scores of the tokens 4 n + i (one page per lane) for the heads 4 b + r
    float4_t sc[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) sc[i] = float4_t{0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < D / 32; ++s) {
      half8_t k[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) k[i] = signed_half8(w.kw[2 * s][i], w.kw[2 * s + 1][i]);
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ql[s], k[i], sc[i], 0, 0, 0);
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(qh[s], k[i], sc[i], 0, 0, 0);
    }
    bad |= w.codec != CF_KV_CODEC_INT8 || w.dim != D;
    // tokens of a page are visible from its first on
    const uint32_t page = 16 * (n >> 2), here = visible - 64 * g;  // g is a visible group
    const uint32_t end = min(page + min(w.tc, 16u), here);         // of the page, in tokens of the group
    bool page_vis = w.tc > 0 && page < here;                       // and its V not all 0, as far as that is looked at
    const float ks = w.ks, vs = w.vs;
    // exponent of the group's largest V scale among its visible pages, less 15 (see below)
    constexpr int kNone = -(1 << 24);
    int ep = page_vis && vs != 0.0f ? __builtin_amdgcn_frexp_expf(vs) - 15 : kNone;
    int eb = max(max(__builtin_amdgcn_readlane(ep, 0), __builtin_amdgcn_readlane(ep, 4)),
                 max(__builtin_amdgcn_readlane(ep, 8), __builtin_amdgcn_readlane(ep, 12)));
    // Scales far apart: pages whose visible V are all 0 (their scale is 1, or anything) are left out, lest the others'
    // weights lose their bits to units that nothing needs. (Here, where K's registers are free: behind the softmax's maximum
    // the kernels for whole rows spill, 46.3 -> 53.6 us for 248 rows of 64 listed groups.)
    if (__builtin_amdgcn_ballot_w64(ep < eb - 8 && ep != kNone)) [[unlikely]] {
      const int seen = __shfl(static_cast<int>(max(end, page) - page), 4 * b);  // visible tokens of page b, whose V this lane has
      uint32_t any = 0;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < kTiles; ++i) word |= w.vw[q * kTiles + i] ^ 0x80808080u;
        any |= word & (~0u >> min(max(32 - 8 * (seen - 4 * q), 0), 31)) & (seen > 4 * q ? ~0u : 0u);  // of its visible tokens
      }
      const uint64_t live = __builtin_amdgcn_ballot_w64(any != 0);
      if ((live >> (16 * (n >> 2)) & 0xFFFFu) == 0 && fabsf(vs) < INFINITY) page_vis = false, ep = kNone;
      eb = max(max(__builtin_amdgcn_readlane(ep, 0), __builtin_amdgcn_readlane(ep, 4)),
               max(__builtin_amdgcn_readlane(ep, 8), __builtin_amdgcn_readlane(ep, 12)));
    }
    if (next) w.load_k(next);
    // ---- online softmax
    float p[GT][4], mx[4], sum[4];
    Spread<GT>::deal(sc, p);
    bool moved = false;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float f = unit[r];
      f *= ks;
#pragma unroll
      for (int j = 0; j < GT; ++j) p[j][r] = static_cast<uint32_t>(Spread<GT>::token(n, b, j)) < end ? p[j][r] * f : -INFINITY;
      mx[r] = p[0][r];
#pragma unroll
      for (int j = 1; j < GT; ++j) mx[r] = fmaxf(mx[r], p[j][r]);
    }
    Spread<GT>::reduce_max(mx);
#pragma unroll
    for (int r = 0; r < 4; ++r) moved |= mx[r] > m[r];
    // units of the P.V sums: the exponent of the group's largest V scale among its visible pages, less 15, so that
    // weights p vs lie in [0, 2^15) and those down to 2^-29 of that are normal f16 numbers. Sums move to a larger unit
    // at once (a factor of a power of two) and to a smaller one when 2^8 below: then weights down to 2^-21 of the group's
    // largest are normal.
    // 2^31 tokens of weights below 2^15 and symbols up to 2^7 add up to less than 2^53 of the largest unit so far, `top`: in
    // a unit down to 2^-kDrop of it they stay finite. For a smaller one, the sums as they are say how far it may fall.
    constexpr int kSum = 53, kDrop = 60;
    int e_new = e;
    if (eb != kNone && (eb > e || eb < e - 8)) e_new = eb;
    top = max(top, e_new);
    if (__builtin_amdgcn_ballot_w64(moved) || e_new != e) {
      float f[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float mn = fmaxf(m[r], mx[r]);
        f[r] = m[r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[r] - mn);  // 0 before the first visible token
        m[r] = mn;
        l[r] *= f[r];
      }
      if (e_new < top - kDrop) [[unlikely]] {
        float big = 0.0f;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int i = 0; i < kTiles; ++i) {
            acc[i][r] *= f[r];
            if (static_cast<uint32_t>(4 * b + r) < gqa) big = fmaxf(big, fabsf(acc[i][r]));  // (other rows hold anything)
          }
        big = cfd::rows4_max(cfd::row16_max(big));
        top = big > 0.0f ? max(e_new, __builtin_amdgcn_readfirstlane(__builtin_amdgcn_frexp_expf(big)) + e - kSum) : e_new;
        e_new = max(e_new, top - kDrop);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int i = 0; i < kTiles; ++i) acc[i][r] = ldexpf(acc[i][r], e - e_new);
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          f[r] = ldexpf(f[r], max(e - e_new, -200));
#pragma unroll
          for (int i = 0; i < kTiles; ++i) acc[i][r] *= f[r];
        }
      }
      e = e_new;
    }
    const float vsn = page_vis ? ldexpf(vs, -e) : 0.0f;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float m0 = m[r] == -INFINITY ? 0.0f : m[r];
#pragma unroll
      for (int j = 0; j < GT; ++j) p[j][r] = __builtin_amdgcn_exp2f(p[j][r] - m0);  // exp2(-inf) = 0
      sum[r] = p[0][r];
#pragma unroll
      for (int j = 1; j < GT; ++j) sum[r] += p[j][r];
      l[r] += sum[r];
    }
    if (stats) {
      Spread<GT>::reduce_sum(sum);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (n == r && b < GT && static_cast<uint32_t>(4 * b + r) < gqa) put(4 * b + r, m[r], sum[r]);
    }
    if (Spread<GT>::head(b, 0) < gqa) {
      const int at = Spread<GT>::token(n, b, 0);
      if constexpr (GT == 1) {
        _Float16 h[4], lo[4];
        cfd::split2_mul_f16(p[0][0], p[0][1], vsn, h[0], lo[0], h[1], lo[1]);
        cfd::split2_mul_f16(p[0][2], p[0][3], vsn, h[2], lo[2], h[3], lo[3]);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          lds.p[0][r][at] = h[r];
          lds.p[1][r][at] = lo[r];
        }
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          _Float16 h[GT], lo[GT];
#pragma unroll
          for (int j = 0; j < GT; j += 2) cfd::split2_mul_f16(p[j][r], p[j + 1][r], vsn, h[j], lo[j], h[j + 1], lo[j + 1]);
          typedef _Float16 halves_t __attribute__((ext_vector_type(GT)));
          halves_t hv, lv;
#pragma unroll
          for (int j = 0; j < GT; ++j) hv[j] = h[j], lv[j] = lo[j];
          *reinterpret_cast<halves_t *>(&lds.p[0][Spread<GT>::head(b, r)][at]) = hv;
          *reinterpret_cast<halves_t *>(&lds.p[1][Spread<GT>::head(b, r)][at]) = lv;
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    // ---- P.V: k-values of lane group b = tokens 8 tp .. 8 tp + 7 of page b
#pragma unroll
    for (int tp = 0; tp < 2; ++tp) {
      const half8_t ph = *reinterpret_cast<const half8_t *>(&lds.p[0][n][16 * b + 8 * tp]);
      const half8_t pl = *reinterpret_cast<const half8_t *>(&lds.p[1][n][16 * b + 8 * tp]);
#pragma unroll
      for (int i0 = 0; i0 < kTiles; i0 += 4) {
        half8_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = signed_half8(w.vw[2 * tp * kTiles + i0 + i], w.vw[(2 * tp + 1) * kTiles + i0 + i]);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i0 + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pl, v[i], acc[i0 + i], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i0 + i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph, v[i], acc[i0 + i], 0, 0, 0);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    if (next) w.load_v(next);
  }

  // l becomes the sum over all lanes; m a NaN where the row is broken or holds one (a NaN score leaves the maximum as it was
  // and makes the sum a NaN). attended: whether a group was. Where every score was -inf, l is then 1 beside the maximum of -inf:
  // unlike a state without a token, it makes a row NaN that has nothing else.
  __device__ __forceinline__ void close(bool attended) {
    const bool broken = __builtin_amdgcn_ballot_w64(bad) != 0;
    Spread<GT>::reduce_sum(l);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (attended && m[r] == -INFINITY && l[r] == 0.0f) l[r] = 1.0f;
      if (broken || l[r] != l[r]) m[r] = __builtin_nanf("");
    }
  }

  // The closed state to memory, its sums in absolute units.
  __device__ __forceinline__ void store(float *sums, float2 *states, uint32_t gqa) const {
    const int lane = threadIdx.x & 63, n = lane & 15, b = lane >> 4;
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (static_cast<uint32_t>(4 * b + r) < gqa) {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) sums[(4 * b + r) * D + 16 * i + n] = ldexpf(acc[i][r], max(e, -200));
        if (n == 0) states[4 * b + r] = float2{m[r], l[r]};
      }
  }
};

__device__ __forceinline__ const uint8_t *blob_at(const SelArgs &a, uint32_t offsets, int lane) {
  // (readlane returns an int: offsets from 2^31 on must not be sign-extended)
  return a.d.pool + static_cast<size_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(offsets, lane))) * 16;
}

// Statistics of `count` slots looked up together from the wavefront's LDS to memory; `dest`: the place of this lane's slot.
__device__ __forceinline__ void write_stats(float2 *__restrict__ to, const float2 *stat, uint32_t dest, uint32_t count,
                                            uint32_t gqa) {
  const uint32_t lane = threadIdx.x & 63;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  for (uint32_t e0 = 0; e0 < count * gqa; e0 += 64) {
    const uint32_t e = e0 + lane, i = min(e / gqa, 63u);
    const size_t at = __shfl(dest, static_cast<int>(i));
    if (e < count * gqa) to[at * gqa + (e - i * gqa)] = stat[e];
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// kRow and kSplit: a workgroup takes slots of one row, its wavefronts a block of them each.
template <int D, int W, bool ROW, int GT>
__global__ __launch_bounds__(64 * W, 2) void row_kernel(SelArgs a) {
  __shared__ union {
    WaveLds wave[W];
    float red[W][kRows][D];
  } sh;
  __shared__ float s_m[W][kRows], s_l[W][kRows];
  __shared__ float s_top[kRows], s_inv[kRows];
  __shared__ float2 s_stat[ROW ? kRowStats : 1];

  const int lane = threadIdx.x & 63, n = lane & 15, b = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t head = blockIdx.y, seq = blockIdx.z;
  const uint32_t gqa = a.d.query_head_count / a.d.kv_head_count;
  const size_t row = static_cast<size_t>(seq) * a.d.kv_head_count + head;
  // Workgroups go to the 8 dies in turn: with a multiple of 8 splits a die would take the same splits of every row, and the
  // last ones are empty in short rows (32 x 500-32768 tokens in 8 splits: 278 us, rotated 222).
  const uint32_t split = ROW ? 0 : (blockIdx.x + static_cast<uint32_t>(row % a.splits)) % a.splits;
  const uint32_t *list = a.s.units ? a.s.units + row * a.s.max_units : nullptr;
  const uint32_t *grow = a.d.group_offsets + row * a.d.max_groups;
  // The queries' loads come first, so that they are there when the list entry and the offset, which the first group waits
  // for anyway, have come.
  Query<D> q;
  q.load(a, seq, head, gqa);
  const uint32_t visible = visible_tokens(a.d.seq_tokens[seq], a.d.query_pos[seq], a.d.max_groups);
  const uint32_t ngroups = (visible + 63) / 64, nslots = row_slots(a, ngroups);
  const uint32_t s0 = ROW ? 0 : min(split * a.per, nslots), s1 = ROW ? nslots : min(nslots, s0 + a.per);
  RowState<D, GT> st;
  st.reset();
  bool split_done = false, bad = false;
  // Slots are looked up 64 at a time (fewer where that many statistics would not fit), one a lane, so that no load of the
  // loop below waits for a list entry or an offset.
  const uint32_t pw = (s1 - s0 + W - 1) / W, w0 = min(s1, s0 + wave * pw), w1 = min(s1, w0 + pw);
  const uint32_t step = ROW ? 64u : look_slots(gqa);
  const bool stats = a.s.weights_out != nullptr;
  WaveLds &lds = sh.wave[wave];
  for (uint32_t c0 = w0; c0 < w1; c0 += step) {
    const uint32_t mine = c0 + lane;
    float2 *stat = ROW ? s_stat + c0 * gqa : lds.stat;
    uint32_t g_l = 0xFFFFFFFFu, off_l = 0;
    const bool in = mine < w1 && static_cast<uint32_t>(lane) < step;
    if (in) {
      g_l = listed_group(a, list, mine, bad);
      if (g_l < ngroups) off_l = grow[g_l];
    }
    const bool here = g_l < ngroups;
    uint64_t todo = __builtin_amdgcn_ballot_w64(here);
    if (stats && in && !here)
      for (uint32_t h = 0; h < gqa; ++h) stat[lane * gqa + h] = float2{-INFINITY, 0.0f};
    if (todo) {
      int cur = __builtin_ctzll(todo);
      Blob<D> w;
      w.load_k(blob_at(a, off_l, cur));
      w.load_v(blob_at(a, off_l, cur));
      if (!split_done) st.set_query(a, q, gqa);
      split_done = true;
      for (;;) {
        todo &= todo - 1;
        const int next = todo ? __builtin_ctzll(todo) : -1;
        const uint32_t g = static_cast<uint32_t>(__builtin_amdgcn_readlane(g_l, cur));
        float2 *put = stat + static_cast<uint32_t>(cur) * gqa;
        st.attend(w, g, visible, gqa, lds, next >= 0 ? blob_at(a, off_l, next) : nullptr, stats,
                  [&](uint32_t h, float m, float l) { put[h] = float2{m, l}; });
        if (next < 0) break;
        cur = next;
      }
    }
    if (!ROW && stats) write_stats(a.stats + row * a.slots * gqa, lds.stat, mine, min(step, w1 - c0), gqa);
  }
  st.bad |= bad;
  st.close(!ROW && split_done);
  // ---- join the wavefronts
  if (n == 0) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      s_m[wave][4 * b + r] = st.m[r];
      s_l[wave][4 * b + r] = st.l[r];
    }
  }
  __syncthreads();  // (and the wavefronts' areas are dead)
  if (static_cast<uint32_t>(4 * b) < gqa) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < D / 16; ++i) sh.red[wave][4 * b + r][16 * i + n] = ldexpf(st.acc[i][r], max(st.e, -200));
  }
  __syncthreads();
  const size_t at = (row * a.splits + split) * gqa;
  for (uint32_t i = threadIdx.x; i < gqa * D; i += 64 * W) {
    const uint32_t h = i / D, dd = i % D;
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    bool nan = false;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      nan |= s_m[w][h] != s_m[w][h];
      m = fmaxf(m, s_m[w][h]);
    }
    if (m != -INFINITY)
#pragma unroll
      for (int w = 0; w < W; ++w) {
        if (s_m[w][h] == -INFINITY) continue;
        const float f = __builtin_amdgcn_exp2f(s_m[w][h] - m);
        l += s_l[w][h] * f;
        o += sh.red[w][h][dd] * f;
      }
    if constexpr (ROW) {  // lists ascend: the first entry is visible if any is
      if (m == -INFINITY && nslots) nan |= listed_group(a, list, 0, bad) < ngroups;
    } else if (m == -INFINITY) {
#pragma unroll
      for (int w = 0; w < W; ++w) l += s_l[w][h];  // (not 0 where all scores are -inf: see close())
    }
    if (nan) m = __builtin_nanf("");
    if constexpr (ROW) {
      a.d.output[(static_cast<size_t>(seq) * a.d.query_head_count + head * gqa + h) * D + dd] =
          nan ? m : m == -INFINITY ? 0.0f : o / l;
      if (dd == 0) {
        s_top[h] = m;
        s_inv[h] = 1.0f / l;
      }
    } else {
      a.sums[at * D + i] = o;
      if (dd == 0) a.states[at + h] = float2{m, l};
    }
  }
  if constexpr (ROW) {
    if (!a.s.weights_out) return;
    __syncthreads();
    write_weights(a, row, list, ngroups, nslots, 0, a.d.max_groups, gqa, s_top, s_inv,
                  [&](uint32_t slot, uint32_t h) { return s_stat[slot * gqa + h]; });
  }
}

// Stretches of `total` slots over nwaves wavefronts: the first total % nwaves of them one slot longer.
struct Stretch {
  uint32_t q, r;
  __device__ Stretch(uint32_t total, uint32_t nwaves) : q(total / nwaves), r(total % nwaves) {}
  __device__ uint32_t begin(uint32_t j) const { return j * q + min(j, r); }
  __device__ uint32_t owner(uint32_t x) const { return x < r * (q + 1) ? x / (q + 1) : r + (x - r * (q + 1)) / q; }
};

// kSpan. A wavefront's stretch touches consecutive rows; it leaves one state for each of them, number wavefront + row in
// the laid-out order (head * seq_count + sequence), which no other wavefront has, and a row's states lie side by side.
template <int D, int GT>
__global__ __launch_bounds__(64 * kWaves, 2) void span_kernel(SelArgs a) {
  constexpr int T = 64 * kWaves;
  __shared__ WaveLds s_wave[kWaves];
  __shared__ uint32_t s_pre[kSpanSeqs + 1], s_vis[kSpanSeqs], s_tot[kWaves];
  const uint32_t tid = threadIdx.x, S = a.d.seq_count, lane = tid & 63;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const uint32_t gqa = a.d.query_head_count / a.d.kv_head_count;
  uint32_t base = 0;
  for (uint32_t c = 0; c < S; c += T) {
    const uint32_t s = c + tid;
    uint32_t n = 0, total;
    if (s < S) {
      const uint32_t vis = visible_tokens(a.d.seq_tokens[s], a.d.query_pos[s], a.d.max_groups);
      n = row_slots(a, (vis + 63) / 64);
      s_vis[s] = vis;
    }
    uint32_t before = base + cfsel::wave_prefix(n, total);
    if (c) __syncthreads();
    if (lane == 0) s_tot[wave] = total;
    __syncthreads();
    for (uint32_t w = 0; w < kWaves; ++w) {
      if (w < wave) before += s_tot[w];
      base += s_tot[w];
    }
    if (s < S) s_pre[s] = before;
  }
  if (tid == 0) s_pre[S] = base;
  __syncthreads();
  const uint32_t per_head = base;
  if (blockIdx.x == 0)
    for (uint32_t i = tid; i <= S; i += T) a.pre[i] = s_pre[i];
  const uint32_t me = blockIdx.x * kWaves + wave;
  if (me >= a.nwaves) return;
  const Stretch part(per_head * a.d.kv_head_count, a.nwaves);
  const uint32_t x0 = part.begin(me), x1 = part.begin(me + 1), step = look_slots(gqa);
  const bool stats = a.s.weights_out != nullptr;
  if (x0 >= x1) return;
  WaveLds &lds = s_wave[wave];

  // Lane i looks up slot x + i of the stretch: its row, group and blob.
  struct Look {
    uint32_t row, g, off, dest, vis;  // dest: the place of the slot's statistics
    bool here, bad;
  };
  auto look = [&](uint32_t x) {
    Look k{};
    const uint32_t y = x + lane;
    k.g = 0xFFFFFFFFu;
    k.here = false;
    k.bad = false;
    if (y < x1 && lane < step) {
      const uint32_t head = y / per_head, z = y - head * per_head;
      uint32_t lo = 0, hi = S;  // the last sequence that begins at or before z: one that holds it
      while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2;
        if (s_pre[mid] <= z) lo = mid;
        else hi = mid;
      }
      k.row = head * S + lo;
      const uint32_t slot = z - s_pre[lo];
      k.vis = s_vis[lo];
      const size_t r = static_cast<size_t>(lo) * a.d.kv_head_count + head;
      k.dest = static_cast<uint32_t>(r) * a.slots + slot;
      k.g = listed_group(a, a.s.units ? a.s.units + r * a.s.max_units : nullptr, slot, k.bad);
      k.here = k.g < (k.vis + 63) / 64;
      if (k.here) k.off = a.d.group_offsets[r * a.d.max_groups + k.g];
      else if (stats)
        for (uint32_t h = 0; h < gqa; ++h) lds.stat[lane * gqa + h] = float2{-INFINITY, 0.0f};
    }
    return k;
  };
  auto lane_of = [](uint32_t x, int i) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(x, i)); };

  RowState<D, GT> st;
  st.reset();
  Blob<D> w;
  Look k{};
  uint32_t x = x0 - step, row = 0, q_row = 0xFFFFFFFFu;
  uint64_t todo = 0;
  bool first = true, in_flight = false;
  auto row_broken = [&] { return __builtin_amdgcn_ballot_w64(k.bad && k.row == row) != 0; };
  for (;;) {
    const bool group = todo != 0;
    const int cur = group ? __builtin_ctzll(todo) : static_cast<int>(min(step, x1 - x) - 1);
    const bool done = !group && !first && x + step >= x1;
    if (!group && !first && stats) write_stats(a.stats, lds.stat, k.dest, min(step, x1 - x), gqa);
    // rows up to the one at hand are closed; those without a group in this stretch leave an empty state
    const uint32_t r = lane_of(k.row, cur) + (done ? 1u : 0u);
    if (!first)
      for (; row != r; ++row) {
        st.bad |= row_broken();
        st.close(q_row == row);
        const size_t state = static_cast<size_t>(me) + row;
        st.store(a.sums + state * gqa * D, a.states + state * gqa, gqa);
        st.reset();
      }
    if (done) break;
    if (!group) {  // the next slots
      if (!first) st.bad |= row_broken();
      x += step;
      k = look(x);
      todo = __builtin_amdgcn_ballot_w64(k.here);
      if (first) row = lane_of(k.row, 0);
      first = false;
      in_flight = false;
      continue;
    }
    if (!in_flight) {
      w.load_k(blob_at(a, k.off, cur));
      w.load_v(blob_at(a, k.off, cur));
      in_flight = true;
    }
    const uint32_t seq = row % S, head = row / S;
    if (q_row != row) {
      Query<D> q;
      q.load(a, seq, head, gqa);
      st.set_query(a, q, gqa);
      q_row = row;
    }
    todo &= todo - 1;
    const uint8_t *next = todo ? blob_at(a, k.off, __builtin_ctzll(todo)) : nullptr;
    float2 *put = lds.stat + static_cast<uint32_t>(cur) * gqa;
    st.attend(w, lane_of(k.g, cur), lane_of(k.vis, cur), gqa, lds, next, stats,
              [&](uint32_t h, float m, float l) { put[h] = float2{m, l}; });
  }
}

// ---- RANS_HYBRID pools: the batched decode's group body (kv_group_body.hpp; at most 4 query heads per KV head), groups of a
// unit decoded back to back by one wavefront, since a chain may run across them. Bound by the entropy decode, as there: the
// tables are staged by every workgroup and the memory pipeline restarts at every row. 32 pairs of 512 groups for each of
// 32 x 8 rows (252 MB) 67 us, all their 512 groups (2.02 GB) 482, 468 without weights (kv_batched.hip 374). Two
// wavefronts a SIMD: at three the code for raw groups beside the lookups spills (81 and 484 us with 13 registers spilled,
// 111 and 622 with 58).

// A unit's groups in this launch: the list's units, or pairs (a chain never spans more).
__host__ __device__ inline uint32_t coded_item(const cf_kv_selection &s) { return s.units ? s.unit_groups : 2u; }

template <int D>
__global__ __attribute__((amdgpu_waves_per_eu(2, 8))) __launch_bounds__(64 * kWaves) void coded_kernel(SelArgs a) {
  using namespace cfkv;
  constexpr int W = kWaves, NQ = D / 4, RAW = raw_words<D>(), BUF = buf_u32<D>(), T = 64 * W;
  __shared__ __attribute__((aligned(16))) uint2 s_tab[2][kSlots];
  __shared__ __attribute__((aligned(16))) _Float16 s_p[W][2][4][kGqa][16];
  __shared__ uint32_t s_buf[W][BUF];  // per wavefront: staged words; query staging and the joined states alias it
  static_assert(2 * kGqa * D * 2 <= W * BUF * 4, "query staging must fit the word buffers");
  const int lane = threadIdx.x & 63, G = lane >> 4, t = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t head = blockIdx.y, seq = blockIdx.z;
  const uint32_t gqa = a.d.query_head_count / a.d.kv_head_count;
  const size_t row = static_cast<size_t>(seq) * a.d.kv_head_count + head;
  const uint32_t split = (blockIdx.x + static_cast<uint32_t>(row % a.splits)) % a.splits;  // (see row_kernel)
  const uint32_t *list = a.s.units ? a.s.units + row * a.s.max_units : nullptr;
  const uint32_t *grow = a.d.group_offsets + row * a.d.max_groups;
  const uint32_t visible = visible_tokens(a.d.seq_tokens[seq], a.d.query_pos[seq], a.d.max_groups);
  const uint32_t ngroups = (visible + 63) / 64, nslots = row_slots(a, ngroups), item = coded_item(a.s);
  const uint32_t s0 = min(split * a.per, nslots), s1 = min(nslots, s0 + a.per);

  // ---- tables and queries, as kv_batched_kernel stages them
  {
    const uint4 *tk = reinterpret_cast<const uint4 *>(a.d.tables + static_cast<size_t>(2 * head) * CF_KV_RANS_TABLE_BYTES);
    constexpr int kIt = static_cast<int>(kSlots / T);
    static_assert(kSlots % T == 0, "two table entries a thread and step");
    uint4 e[kIt];
#pragma unroll
    for (int k = 0; k < kIt; ++k) e[k] = tk[threadIdx.x + k * T];
#pragma unroll
    for (int k = 0; k < kIt; ++k) {
      const uint32_t j = 2 * (threadIdx.x + k * T);
      *reinterpret_cast<uint4 *>(&s_tab[j / kSlots][j % kSlots]) =
          uint4{(e[k].x & 2047u) | (((e[k].x >> 11) & 2047u) << 16), e[k].y,
                (e[k].z & 2047u) | (((e[k].z >> 11) & 2047u) << 16), e[k].w};
    }
  }
  _Float16(*s_q)[kGqa][D] = reinterpret_cast<_Float16(*)[kGqa][D]>(&s_buf[0][0]);
  for (int i = threadIdx.x; i < kGqa * D; i += T) {
    const int h = i / D, dd = i % D;
    const float q = static_cast<uint32_t>(h) < gqa
                        ? a.d.queries[(static_cast<size_t>(seq) * a.d.query_head_count + head * gqa + h) * D + dd]
                        : 0.0f;
    cfd::split_mul_f16(q, a.d.softmax_scale, s_q[0][h][dd], s_q[1][h][dd]);
  }
  __syncthreads();
  constexpr int NC = NQ / 16 > 0 ? NQ / 16 : 1;
  cfkv::half4_t qhi[NC], qlo[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int qd = 16 * c + (lane >> 2);
    qhi[c] = (4 * qd < D) ? *reinterpret_cast<const cfkv::half4_t *>(&s_q[0][lane & 3][4 * qd]) : cfkv::half4_t{0, 0, 0, 0};
    qlo[c] = (4 * qd < D) ? *reinterpret_cast<const cfkv::half4_t *>(&s_q[1][lane & 3][4 * qd]) : cfkv::half4_t{0, 0, 0, 0};
  }
  float qsum[kGqa];
  {
    float part = 0.0f;
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
      part += static_cast<float>(s_q[0][G][t * (D / 16) + k]) + static_cast<float>(s_q[1][G][t * (D / 16) + k]);
    part = cfd::row16_sum(part);
#pragma unroll
    for (int h = 0; h < kGqa; ++h) qsum[h] = __shfl(part, 16 * h);
  }
  __syncthreads();  // s_q is dead from here on

  float m_run[kGqa], l_run[kGqa];
  VUnit<true> unit;
  cfkv::float4_t acc_v[D / 16];
#pragma unroll
  for (int h = 0; h < kGqa; ++h) m_run[h] = -INFINITY, l_run[h] = 0.0f;
#pragma unroll
  for (int i = 0; i < D / 16; ++i) acc_v[i] = cfkv::float4_t{0, 0, 0, 0};

  uint32_t *buf = s_buf[wave];
  const bool stats = a.s.weights_out != nullptr;
  bool bad = false;  // a list that does not ascend, or a group that continues a chain its unit does not begin
  bool attended = false;
  // blocks of whole units for the wavefronts; slots are looked up 64 at a time, one a lane
  const uint32_t items = (s1 - s0 + item - 1) / item, pw = (items + W - 1) / W * item;
  const uint32_t w0 = min(s1, s0 + wave * pw), w1 = min(s1, w0 + pw);
  for (uint32_t c0 = w0; c0 < w1; c0 += 64) {
    const uint32_t mine = c0 + lane;
    uint32_t g_l = 0xFFFFFFFFu, off_l = 0;
    if (mine < w1) {
      g_l = listed_group(a, list, mine, bad);
      if (g_l < ngroups) off_l = grow[g_l];
    }
    const bool here = g_l < ngroups;
    uint64_t todo = __builtin_amdgcn_ballot_w64(here);
    float2 stat[kGqa];  // of this lane's slot
#pragma unroll
    for (int h = 0; h < kGqa; ++h) stat[h] = float2{-INFINITY, 0.0f};
    if (todo) {
      // The memory pipeline is kv_batched_kernel's: the next group's header and chain states at the start of a group, its word
      // streams into the wavefront's LDS after the decode, its first raw words as the last of this group's are used up.
      uint32_t h_cnt = 0, h_chain = 0, h_tc = 0, h_codec = 0, h_st[2] = {0, 0};
      float h_ks = 0.f, h_vs = 0.f;
      auto load_header = [&](const uint8_t *p) {
        h_st[0] = reinterpret_cast<const uint32_t *>(p + cfkv::kHdr)[lane];
        h_st[1] = reinterpret_cast<const uint32_t *>(p + cfkv::kHdr)[64 + lane];
        h_cnt = *reinterpret_cast<const uint32_t *>(p + 4);
        h_chain = *reinterpret_cast<const uint16_t *>(p + 8);
        h_tc = reinterpret_cast<const uint16_t *>(p + 12)[G];
        h_ks = reinterpret_cast<const float *>(p + 32)[G];
        h_vs = reinterpret_cast<const float *>(p + 48)[G];
        h_codec = *reinterpret_cast<const uint32_t *>(p);
      };
      auto raw_of = [&](const uint8_t *p, uint32_t chain) {
        return reinterpret_cast<const uint32_t *>(p + cfkv::kHdr + (chain ? kStateBytes : 0));
      };
      constexpr int kStage16 = ((kCapWords * 2) + 1023) / 1024;
      auto stage_words = [&](const uint8_t *p, uint32_t chain, uint32_t cnt) {
        const uint32_t nbytes = ((min((cnt & 0xFFFFu) + (cnt >> 16), kCapWords) * 2u) + 15u) & ~15u;
        const uint8_t *src = reinterpret_cast<const uint8_t *>(raw_of(p, chain) + 2 * RAW) + 16u * lane;
#pragma unroll
        for (int k = 0; k < kStage16; ++k)
          if (1024u * k + 16u * lane < nbytes)
            __builtin_amdgcn_global_load_lds(reinterpret_cast<const uint32_t *>(src + 1024 * k),
                                             (__attribute__((address_space(3))) void *)(buf + 256 * k), 16, 0, 0);
      };
      attended = true;
      int cur = __builtin_ctzll(todo);
      const uint8_t *blob = blob_at(a, off_l, cur);
      load_header(blob);
      uint32_t pre[14];
#pragma unroll
      for (int w = 0; w < 14; ++w) pre[w] = 0;
      if (h_codec == CF_KV_CODEC_RANS_HYBRID) {
        const uint32_t *lw = raw_of(blob, h_chain);
#pragma unroll
        for (int w = 0; w < 7; ++w) {
          pre[w] = lw[w * 64 + lane];
          pre[7 + w] = lw[RAW + w * 64 + lane];
        }
        stage_words(blob, h_chain, h_cnt);
      }
      uint32_t st[2] = {0, 0}, prev = 0xFFFFFFFFu;
      for (;;) {
        const uint32_t gi = static_cast<uint32_t>(__builtin_amdgcn_readlane(g_l, cur));
        const uint32_t cnt = h_cnt, chain = h_chain, tcG = h_tc, gcodec = h_codec;
        const float ks = h_ks, vs = h_vs;
        const uint8_t *here_blob = blob;
        const bool tok_ok = static_cast<uint32_t>(t) < tcG && 64 * gi + 16 * G + t < visible;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this group's words have landed
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (gcodec == CF_KV_CODEC_RANS_HYBRID) {
          if (chain) {
            st[0] = h_st[0];
            st[1] = h_st[1];
          } else {
            bad |= prev + 1 != gi || (c0 + static_cast<uint32_t>(cur)) % item == 0;
          }
        }
        todo &= todo - 1;
        const int next = todo ? __builtin_ctzll(todo) : -1;
        if (next >= 0) {
          blob = blob_at(a, off_l, next);
          load_header(blob);
        }
        const bool next_rans = next >= 0 && h_codec == CF_KV_CODEC_RANS_HYBRID;
        const uint32_t *nlw = next_rans ? raw_of(blob, h_chain) : nullptr;
        auto stage_next = [&]() {
          if (next_rans) stage_words(blob, h_chain, h_cnt);
        };
        float p[kGqa];
        if (gcodec == CF_KV_CODEC_RANS_HYBRID)
          group_body<D, CF_KV_CODEC_RANS_HYBRID, 0, const uint16_t *, decltype(stage_next), false, false, false, true>(
              stage_next, pre, nlw, st, raw_of(here_blob, chain), reinterpret_cast<const uint16_t *>(buf), cnt, s_tab, qhi, qlo,
              qsum, s_p[wave], static_cast<uint32_t *>(nullptr), lane, tok_ok, ks, vs, unit, gqa, m_run, l_run, acc_v,
              static_cast<uint32_t *>(nullptr), false, p);
        else
          group_body<D, CF_KV_CODEC_INT8, 0, const uint16_t *, decltype(stage_next), false, false, false, true>(
              stage_next, pre, nlw, st, reinterpret_cast<const uint32_t *>(here_blob + cfkv::kHdr),
              static_cast<const uint16_t *>(nullptr), 0, s_tab, qhi, qlo, qsum, s_p[wave], static_cast<uint32_t *>(nullptr), lane,
              tok_ok, ks, vs, unit, gqa, m_run, l_run, acc_v, static_cast<uint32_t *>(nullptr), false, p);
        if (stats) {
#pragma unroll
          for (int h = 0; h < kGqa; ++h) {
            const float sum = cfd::rows4_sum(cfd::row16_sum(p[h]));
            if (lane == cur) stat[h] = float2{m_run[h] * kLog2e, sum};
          }
        }
        prev = gi;
        if (next < 0) break;
        cur = next;
      }
    }
    if (stats && mine < w1) {
#pragma unroll
      for (int h = 0; h < kGqa; ++h)
        if (static_cast<uint32_t>(h) < gqa) a.stats[(row * a.slots + mine) * gqa + h] = stat[h];
    }
  }

  // ---- reduce the wavefront and join the workgroup, as kv_batched_kernel does
#pragma unroll
  for (int i = 0; i < D / 16; ++i)
#pragma unroll
    for (int h = 0; h < kGqa; ++h) {
      float v = G < 2 ? ldexpf(acc_v[i][h], unit.e()) : 0.0f;
      v += __shfl_xor(v, 16);
      v += __shfl_xor(v, 32);
      acc_v[i][h] = v;
    }
#pragma unroll
  for (int h = 0; h < kGqa; ++h) l_run[h] = cfd::rows4_sum(cfd::row16_sum(l_run[h]));
  const bool broken = __builtin_amdgcn_ballot_w64(bad) != 0;
  float *red = reinterpret_cast<float *>(buf);
  if (lane < 16) {
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
      for (int h = 0; h < kGqa; ++h) red[h * (D + 2) + t + 16 * i] = acc_v[i][h];
  }
  if (lane == 0) {
#pragma unroll
    for (int h = 0; h < kGqa; ++h) {
      red[h * (D + 2) + D] = broken || l_run[h] != l_run[h] ? __builtin_nanf("") : m_run[h];
      red[h * (D + 2) + D + 1] = attended && m_run[h] == -INFINITY ? 1.0f : l_run[h];  // (see RowState::close)
    }
  }
  __syncthreads();
  const size_t at = (row * a.splits + split) * gqa;
  for (uint32_t i = threadIdx.x; i < gqa * D; i += T) {
    const uint32_t h = i / D, dd = i % D;
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    bool nan = false;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float mw = reinterpret_cast<const float *>(s_buf[w])[h * (D + 2) + D];
      nan |= mw != mw;
      m = fmaxf(m, mw);
    }
    if (m != -INFINITY)
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float *rw = reinterpret_cast<const float *>(s_buf[w]) + h * (D + 2);
        if (rw[D] == -INFINITY) continue;
        const float f = __builtin_amdgcn_exp2f((rw[D] - m) * kLog2e);
        l += rw[D + 1] * f;
        o += rw[dd] * f;
      }
    else
#pragma unroll
      for (int w = 0; w < W; ++w) l += reinterpret_cast<const float *>(s_buf[w])[h * (D + 2) + D + 1];
    a.sums[at * D + i] = o;
    if (dd == 0) a.states[at + h] = float2{nan ? __builtin_nanf("") : m * kLog2e, l};
  }
}

constexpr int kJoinThreads = 512;
constexpr uint32_t kJoinGroups = 1024;  // groups whose weights one workgroup writes
constexpr uint32_t kFewStates = 16;     // states of a row up to which one workgroup makes the outputs of all its heads

// Joins a row's states: grid (KV heads, sequences, `outs` + parts of the weights). The first `outs` workgroups of a row make its
// outputs: one of them all query heads' (few states a row: 256 rows of 9, 6.5 against 10.5 us with one for each head), or
// one each (many: the states are dealt out over the threads). The others turn group statistics into weights, kJoinGroups
// groups each. Values of many states are loaded at a time: the caches of other dies hold them, so that each load takes about
// a microsecond.
template <int D, bool SPAN>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(SelArgs a, uint32_t outs) {
  constexpr uint32_t kB = 8;
  __shared__ float s_m[kRows], s_inv[kRows];
  __shared__ float s_o[kJoinThreads];
  const uint32_t head = blockIdx.x, seq = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const uint32_t gqa = a.d.query_head_count / a.d.kv_head_count;
  const size_t row = static_cast<size_t>(seq) * a.d.kv_head_count + head;
  size_t state0 = row * a.splits;
  uint32_t states = a.splits;
  if constexpr (SPAN) {
    const uint32_t per_head = a.pre[a.d.seq_count], at = a.pre[seq], len = a.pre[seq + 1] - at;
    states = 0;
    if (len) {
      const Stretch part(per_head * a.d.kv_head_count, a.nwaves);
      const uint32_t x = head * per_head + at, j = part.owner(x);
      states = part.owner(x + len - 1) - j + 1;
      state0 = static_cast<size_t>(j) + static_cast<size_t>(head) * a.d.seq_count + seq;
    } else {
      state0 = 0;
    }
  }
  const float2 *st = a.states + state0 * gqa;
  const bool out = blockIdx.z < outs, every = !out || outs == 1;  // every: the maxima of all heads are needed
  // Elements [e0, e0 + en) of the row's gqa x D outputs are this workgroup's, `parts` threads an element, each every
  // parts-th state.
  const uint32_t e0 = every ? 0 : blockIdx.z * D, en = every ? gqa * D : D, parts = every ? 1 : kJoinThreads / D;
  const uint32_t part = every ? 0 : tid / D;
  const float *sums = a.sums + state0 * gqa * D;
  // the sums of this thread's first states, in flight while the maxima are found
  float o8[kB];
#pragma unroll
  for (uint32_t u = 0; u < kB; ++u) {
    const uint32_t e = e0 + (every ? min(tid, en - 1) : tid % D);
    o8[u] = out && states ? sums[static_cast<size_t>(min(part + u * parts, states - 1)) * gqa * D + e] : 0.0f;
  }
  // a wavefront per query head: its maximum and the inverse of its sum
  for (uint32_t h = every ? tid >> 6 : blockIdx.z; h < (every ? gqa : blockIdx.z + 1); h += kJoinThreads / 64) {
    float m = -INFINITY, l = 0.0f;
    bool nan = false, low = false;  // low: a state whose scores were all -inf
    for (uint32_t s = lane; s < states; s += 64) {
      const float2 x = st[static_cast<size_t>(s) * gqa + h];
      nan |= x.x != x.x;
      low |= x.x == -INFINITY && x.y != 0.0f;
      const float mn = fmaxf(m, x.x);
      if (mn != -INFINITY) {
        l = (m == -INFINITY ? 0.0f : l * __builtin_amdgcn_exp2f(m - mn)) +
            (x.x == -INFINITY ? 0.0f : x.y * __builtin_amdgcn_exp2f(x.x - mn));
        m = mn;
      }
    }
    const float top = cfd::rows4_max(cfd::row16_max(m));
    l = m == -INFINITY ? 0.0f : l * __builtin_amdgcn_exp2f(m - top);
    l = cfd::rows4_sum(cfd::row16_sum(l));
    nan = __builtin_amdgcn_ballot_w64(nan || (top == -INFINITY && low)) != 0;
    if (lane == 0) {
      s_m[h] = nan ? __builtin_nanf("") : top;
      s_inv[h] = 1.0f / l;
    }
  }
  __syncthreads();
  if (out) {
    for (uint32_t i = every ? tid : tid % D; i < en; i += kJoinThreads) {
      const uint32_t e = e0 + i, h = e / D;
      const float m = s_m[h];
      float o = 0.0f;
      if (m != -INFINITY)
        for (uint32_t s = part; s < states; s += kB * parts) {
          float x[kB], f[kB];
#pragma unroll
          for (uint32_t u = 0; u < kB; ++u) {
            const size_t k = static_cast<size_t>(min(s + u * parts, states - 1)) * gqa;
            f[u] = st[k + h].x;
            x[u] = s == part && i < kJoinThreads ? o8[u] : sums[k * D + e];
          }
#pragma unroll
          for (uint32_t u = 0; u < kB; ++u)
            if (s + u * parts < states && f[u] != -INFINITY) o += x[u] * __builtin_amdgcn_exp2f(f[u] - m);
        }
      if (parts > 1) {
        s_o[tid] = o;
        __syncthreads();
        if (part != 0) return;
        for (uint32_t k = 1; k < parts; ++k) o += s_o[k * D + i];
      }
      a.d.output[(static_cast<size_t>(seq) * a.d.query_head_count + head * gqa) * D + e] =
          m != m ? m : m == -INFINITY ? 0.0f : o * s_inv[h];
    }
    return;
  }
  const uint32_t ngroups = (visible_tokens(a.d.seq_tokens[seq], a.d.query_pos[seq], a.d.max_groups) + 63) / 64;
  const uint32_t lo = (blockIdx.z - outs) * kJoinGroups, hi = min(lo + kJoinGroups, a.d.max_groups);
  const float2 *stats = a.stats + row * a.slots * gqa;
  write_weights(a, row, a.s.units ? a.s.units + row * a.s.max_units : nullptr, ngroups, row_slots(a, ngroups), lo, hi, gqa, s_m,
                s_inv, [&](uint32_t slot, uint32_t h) { return stats[static_cast<size_t>(slot) * gqa + h]; });
}

struct Plan {
  Mode mode;
  uint32_t slots, splits, per, nwaves;
  uint64_t pre_bytes, sum_bytes, state_bytes, stat_bytes;
  uint64_t bytes() const { return pre_bytes + sum_bytes + state_bytes + stat_bytes; }
};

uint64_t round16(uint64_t x) { return (x + 15) / 16 * 16; }

Plan make_plan(const cf_kv_batched_desc *d, const cf_kv_selection *s) {
  Plan p{};
  p.slots = s->units ? s->max_units * s->unit_groups : d->max_groups;
  const uint64_t rows = static_cast<uint64_t>(d->seq_count) * d->kv_head_count, all = rows * p.slots;
  const uint32_t gqa = d->query_head_count / d->kv_head_count, cus = cfd::cu_count();
  const bool fits = static_cast<uint64_t>(p.slots) * gqa <= kRowStats;  // a row's statistics in LDS
  uint64_t states = 0;
  // us of a call with weights, 8 KV heads, head_dim 128, 4 query heads per KV head unless said, as kSpan / kRow / kSplit:
  //   32 x 64 of up to 512 groups (list)     55.9 /  47.5 /  53.3      32 x 512 groups            336.4 / 320.7 / 356.7
  //   1 x 32 groups (list)                   13.2 /  19.1 /  12.1      32 x 8..512 groups         179.6 / 229.9 / 209.6
  //   16 x 64 groups, 8 query heads          40.8 /  36.3 /  36.9      1 x 512 groups              29.3 / 184.2 /  21.9
  //   64 x 32 groups                         58.9 /  51.8 /  54.8      1 x 2048 groups             60.3 /   -   /  54.3
  //   64 x 16..125 groups of hd 64           63.9 /  66.3 /  76.7      4 x 2048 groups            163.1 /   -   / 174.0
  //   128 x 32 of 128 groups (list)         103.1 / 103.6 / 102.0      256 x 8..32 groups         139.0 / 144.4 / 135.3
  //   16 query heads: 32 x 64 (list)         64.3 /  57.0 /  68.4      32 x 512 groups            394.0 /   -   / 417.3
  // A row to a workgroup where a list makes the rows alike and they fill the chip once, or where they are many and even out
  // by themselves; stretches from 16 slots a resident wavefront on, where its state is small beside them; else splits.
  if (d->codec == CF_KV_CODEC_RANS_HYBRID) p.mode = kCoded;
  else if (d->splits == 1 && fits) p.mode = kRow;
  else if (d->splits != 0) p.mode = kSplit;
  else if (fits && ((s->units && 4 * rows >= 3 * cus && rows <= cus) || rows >= 2 * cus)) p.mode = kRow;
  else if (d->seq_count <= kSpanSeqs && all >= 16ull * kResident * cus && all < 1u << 31) p.mode = kSpan;
  else p.mode = kSplit;
  if (p.mode == kSplit || p.mode == kCoded) {
    const uint32_t item = p.mode == kCoded ? coded_item(*s) : 1, items = (p.slots + item - 1) / item;
    const uint64_t resident = static_cast<uint64_t>(kResident) * cus;
    uint32_t splits = d->splits;
    if (splits == 0) {  // one resident round of wavefronts where there are few slots, at most 16 slots each
      const uint64_t per_wave = std::min<uint64_t>(16 / item, std::max<uint64_t>(1, rows * items / resident));
      splits = static_cast<uint32_t>((items + per_wave * kWaves - 1) / (per_wave * kWaves));
    }
    splits = std::max<uint32_t>(1, std::min(splits, items));
    p.per = (items + splits - 1) / splits * item;
    p.splits = (p.slots + p.per - 1) / p.per;
    states = rows * p.splits;
  } else if (p.mode == kSpan) {
    p.nwaves = kResident * cus;
    p.pre_bytes = round16((d->seq_count + 1ull) * sizeof(uint32_t));
    states = p.nwaves + rows;
  } else {
    p.splits = 1;
  }
  p.sum_bytes = round16(states * gqa * d->head_dim * sizeof(float));
  p.state_bytes = round16(states * gqa * sizeof(float2));
  p.stat_bytes = s->weights_out && p.mode != kRow ? all * gqa * sizeof(float2) : 0;
  return p;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <int D, int GT>
void launch_cut(const SelArgs &a, Mode mode, hipStream_t s) {
  const uint32_t heads = a.d.kv_head_count, seqs = a.d.seq_count;
  if (mode == kRow) row_kernel<D, kWavesRow, true, GT><<<dim3(1, heads, seqs), 64 * kWavesRow, 0, s>>>(a);
  else if (mode == kSpan) span_kernel<D, GT><<<(a.nwaves + kWaves - 1) / kWaves, 64 * kWaves, 0, s>>>(a);
  else row_kernel<D, kWaves, false, GT><<<dim3(a.splits, heads, seqs), 64 * kWaves, 0, s>>>(a);
}

template <int D>
void launch(const SelArgs &a, Mode mode, hipStream_t s) {
  const uint32_t heads = a.d.kv_head_count, seqs = a.d.seq_count, gqa = a.d.query_head_count / heads;
  if (mode == kCoded) coded_kernel<D><<<dim3(a.splits, heads, seqs), 64 * kWaves, 0, s>>>(a);
  else if (gqa <= 4) launch_cut<D, 1>(a, mode, s);
  else if (gqa <= 8) launch_cut<D, 2>(a, mode, s);
  else launch_cut<D, 4>(a, mode, s);
  if (mode == kRow) return;
  const uint32_t parts = a.s.weights_out ? (a.d.max_groups + kJoinGroups - 1) / kJoinGroups : 0;
  // states of a row: of a span, those of an average one
  const uint64_t states = mode == kSpan ? a.nwaves / (static_cast<uint64_t>(heads) * seqs) + 1 : a.splits;
  const uint32_t outs = states <= kFewStates ? 1 : gqa;
  const dim3 join(heads, seqs, outs + parts);
  if (mode == kSpan) join_kernel<D, true><<<join, kJoinThreads, 0, s>>>(a, outs);
  else join_kernel<D, false><<<join, kJoinThreads, 0, s>>>(a, outs);
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
  if (d->max_groups == 0) return CF_ERR_INVALID_ARGUMENT;
  if (d->max_groups >= 1u << 25) return CF_ERR_UNSUPPORTED;  // 64 * max_groups in 32 bits, join grids in z
  if (s->units) {
    if (s->max_units == 0 || (s->unit_groups != 1 && s->unit_groups != 2)) return CF_ERR_INVALID_ARGUMENT;
    if (s->max_units >= 1u << 25) return CF_ERR_UNSUPPORTED;
  }
  if (!std::isfinite(s->decay) || (s->weights_in && !s->weights_out)) return CF_ERR_INVALID_ARGUMENT;
  return CF_OK;
}

extern "C" uint64_t cf_kv_selected_workspace_bytes(const cf_kv_batched_desc *d, const cf_kv_selection *s) {
  if (cf_kv_validate_selection(d, s) != CF_OK) return 0;
  return make_plan(d, s).bytes();
}

extern "C" cf_status cf_kv_paged_attention_selected_async(const cf_kv_batched_desc *d, const cf_kv_selection *s, void *stream) {
  const cf_status v = cf_kv_validate_selection(d, s);
  if (v != CF_OK) return v;
  const Plan p = make_plan(d, s);
  const uint64_t need = p.bytes();
  if (need && (!d->workspace || d->workspace_bytes < need || !aligned16(d->workspace))) return CF_ERR_INVALID_ARGUMENT;
  char *ws = static_cast<char *>(d->workspace);
  SelArgs a{*d, *s, p.slots, p.splits, p.per, p.nwaves, reinterpret_cast<uint32_t *>(ws),
            reinterpret_cast<float *>(ws + p.pre_bytes), reinterpret_cast<float2 *>(ws + p.pre_bytes + p.sum_bytes),
            reinterpret_cast<float2 *>(ws + p.pre_bytes + p.sum_bytes + p.state_bytes)};
  if (!s->units) a.s.unit_groups = 1;
  const hipStream_t st = cfd::as_stream(stream);
  if (d->head_dim == 128) launch<128>(a, p.mode, st);
  else launch<64>(a, p.mode, st);
  return cfd::launch_status();
}
