// kv_topk.hpp — the k largest of n 32-bit keys by one workgroup, ties to the lower index, emitted in index order
// (kv_select.h: selection of units by score, eviction by weight).
#pragma once

#include "cf_device.hpp"

namespace cfsel {

// Order-preserving map of fp32 to u32: -inf < ... < -0 = +0 < ... < +inf < NaN (any NaN).
__device__ __forceinline__ uint32_t sortable(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}

constexpr uint32_t kBins = 2048;
constexpr uint32_t kFew = 96;   // so few keys are ranked by comparing each with all

template <int T>
struct TopkShared {
  __attribute__((aligned(16))) uint32_t hist[kBins];
  uint32_t wave[2][T / 64][2];
  uint32_t lo, hi, bin, above, count;
};

// Lane moves inside the rows of 16 lanes and between rows by DPP, which keep an LDS round trip per step (ds_bpermute) off
// the picks' dependency chain; lanes without a source get 0.
template <int CTRL, int ROWS = 0xf>
__device__ __forceinline__ uint32_t dpp_or_0(uint32_t x) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, ROWS, 0xf, true));
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_all(uint32_t x) {
  return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(x), CTRL, 0xf, 0xf, false));
}

// Sum of x over the lanes below this one (exclusive) and over the whole wavefront: row_shr 1, 2, 4, 8 inside the rows,
// then row_bcast 15 (into rows 1 and 3) and 31 (into rows 2 and 3).
__device__ __forceinline__ uint32_t wave_prefix(uint32_t x, uint32_t &total) {
  uint32_t s = x;
  s += dpp_or_0<0x111>(s);
  s += dpp_or_0<0x112>(s);
  s += dpp_or_0<0x114>(s);
  s += dpp_or_0<0x118>(s);
  s += dpp_or_0<0x142, 0xa>(s);
  s += dpp_or_0<0x143, 0xc>(s);
  total = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(s), 63));
  return s - x;
}

// Largest x of the wavefront, in every lane.
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  x = max(x, dpp_all<0xb1>(x));
  x = max(x, dpp_all<0x4e>(x));
  x = max(x, dpp_all<0x141>(x));
  x = max(x, dpp_all<0x140>(x));
  const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = max(static_cast<uint32_t>(r[0]), static_cast<uint32_t>(r[1]));
  const auto h = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return max(static_cast<uint32_t>(h[0]), static_cast<uint32_t>(h[1]));
}

// Keys key(i) > 0, i < n; of them [0, first) and [n - last, n) are in whatever their keys; k in all are taken,
// first + last <= k. emit(i, taken, pos) is called by one thread for every i < n, `pos` the number of taken (or, for one
// that is not, of untaken) indices before it. Calls come in rounds of T consecutive indices, all threads together;
// round_end(base, taken_before, taken_in_round) is called by all threads after each round's emits. All T threads call this.
//
// Method: the free keys' range [lo, hi] is cut into 2048 equal bins whose shift follows the range (scores of one row share
// their sign and most of their exponent, so fixed digits would send most keys to one counter), the bin where the count
// from the top reaches what is still needed becomes the next range; at most three rounds for 32 bits, mostly one or two:
// a round ends the search when its bin is needed whole. Up to kFew keys: each is compared with all others, one barrier
// instead of about ten (eviction of one of 65 units, a third of them equal, 8.1 -> 6.0 us; 128 units 7.6 -> 8.2).
template <int T, typename Key, typename Emit, typename RoundEnd>
__device__ __forceinline__ void take_largest(const Key &key, uint32_t n, uint32_t first, uint32_t last, uint32_t k,
                                             TopkShared<T> &sh, const Emit &emit, const RoundEnd &round_end) {
  const uint32_t tid = threadIdx.x;
  const int lane = tid & 63, wave = tid >> 6;
  constexpr int W = T / 64;
  uint32_t lo = 0, hi = 0xFFFFFFFFu, need = 0;
  bool all = true, ties = false;  // all: every index is taken; ties: `need` of the keys equal to lo are
  bool ranked = false, ranked_take = false;
  const uint32_t f0 = min(first, n), f1 = max(f0, n - min(last, n));
  if (k < n) {
    all = false;
    need = k - min(k, first + last);
    if (n <= kFew) {
      ranked = true;
      const bool free = tid >= f0 && tid < f1;
      const uint32_t mine = free ? key(tid) : 0u;  // 0: below every key
      if (tid < kFew) sh.hist[tid] = mine;
      __syncthreads();
      // before this wavefront's indices an equal key counts, behind them it does not; among them it is decided lane by lane
      uint32_t rank = 0;
      auto count = [&](uint32_t from, uint32_t to, auto above) {
        for (uint32_t j = from; j < min(to, n); j += 4) {
          const uint4 x = *reinterpret_cast<const uint4 *>(&sh.hist[j]);
          rank += above(x.x, j) + above(x.y, j + 1) + above(x.z, j + 2) + above(x.w, j + 3);
        }
      };
      const uint32_t w0 = 64u * wave;
      count(0, w0, [&](uint32_t x, uint32_t) { return x >= mine ? 1u : 0u; });
      count(w0, w0 + 64, [&](uint32_t x, uint32_t j) { return x > (j < tid ? mine - 1 : mine) ? 1u : 0u; });
      count(w0 + 64, n, [&](uint32_t x, uint32_t) { return x > mine ? 1u : 0u; });
      ranked_take = free && rank < need;
    } else if (need == 0) {  // nothing but the forced ones: no key reaches the range
      lo = 0xFFFFFFFFu;
      hi = 0xFFFFFFFFu;
      ties = true;
    } else {
      uint32_t mn = 0xFFFFFFFFu, mx = 0;
      for (uint32_t i = f0 + tid; i < f1; i += T) {
        const uint32_t x = key(i);
        mn = min(mn, x);
        mx = max(mx, x);
      }
      mn = ~wave_max(~mn);
      mx = wave_max(mx);
      if (lane == 0) {
        sh.wave[0][wave][0] = mn;
        sh.wave[0][wave][1] = mx;
      }
      __syncthreads();
      lo = 0xFFFFFFFFu;
      hi = 0;
      for (int w = 0; w < W; ++w) {
        lo = min(lo, sh.wave[0][w][0]);
        hi = max(hi, sh.wave[0][w][1]);
      }
      for (;;) {
        const uint32_t range = hi - lo;
        const uint32_t shift = range < kBins ? 0u : 21u - static_cast<uint32_t>(__builtin_clz(range));
        for (uint32_t b = tid; b < kBins; b += T) sh.hist[b] = 0;
        __syncthreads();
        for (uint32_t i = f0 + tid; i < f1; i += T) {
          const uint32_t x = key(i);
          if (x >= lo && x <= hi) atomicAdd(&sh.hist[(x - lo) >> shift], 1u);
        }
        __syncthreads();
        // bins from the top: thread t owns kBins / T of them, thread 0 the highest
        constexpr uint32_t kPer = kBins / T;
        uint32_t own = 0;
#pragma unroll
        for (uint32_t j = 0; j < kPer; ++j) own += sh.hist[kBins - 1 - (tid * kPer + j)];
        uint32_t total;
        uint32_t above = wave_prefix(own, total);
        if (lane == 0) sh.wave[1][wave][0] = total;
        __syncthreads();
        for (int w = 0; w < wave; ++w) above += sh.wave[1][w][0];
        if (above < need && need <= above + own) {
          for (uint32_t j = 0; j < kPer; ++j) {
            const uint32_t b = kBins - 1 - (tid * kPer + j), c = sh.hist[b];
            if (above + c >= need) {
              sh.bin = b;
              sh.above = above;
              sh.count = c;
              break;
            }
            above += c;
          }
        }
        __syncthreads();
        const uint32_t bin = sh.bin, cnt = sh.count;
        need -= sh.above;
        lo += bin << shift;
        const uint32_t width = (1u << shift) - 1u;
        if (hi - lo > width) hi = lo + width;
        if (cnt == need) break;  // the whole bin: every key from lo on
        if (shift == 0) {
          ties = true;
          break;
        }
      }
    }
  }
  uint32_t taken0 = 0, eq0 = 0;
  int buf = 0;
  __syncthreads();
  for (uint32_t base = 0; base < n; base += T, buf ^= 1) {
    const uint32_t i = base + tid;
    const bool in = i < n, forced = in && (i < f0 || i >= f1);
    bool take = in && (all || forced || ranked_take), eq = false;
    if (in && !take && !ranked) {
      const uint32_t x = key(i);
      if (ties) {
        take = x > lo;
        eq = x == lo && need != 0;
      } else {
        take = x >= lo;
      }
    }
    const uint64_t me = __builtin_amdgcn_ballot_w64(eq);
    const uint64_t below = (uint64_t(1) << lane) - 1;
    if (lane == 0) sh.wave[buf][wave][1] = static_cast<uint32_t>(__builtin_popcountll(me));
    if (ties) {  // equal keys: the first `need` in index order
      __syncthreads();
      uint32_t rank = eq0 + static_cast<uint32_t>(__builtin_popcountll(me & below));
      for (int w = 0; w < wave; ++w) rank += sh.wave[buf][w][1];
      for (int w = 0; w < W; ++w) eq0 += sh.wave[buf][w][1];
      take |= eq && rank < need;
    }
    const uint64_t mt = __builtin_amdgcn_ballot_w64(take);
    if (lane == 0) sh.wave[buf][wave][0] = static_cast<uint32_t>(__builtin_popcountll(mt));
    __syncthreads();
    uint32_t pos = taken0 + static_cast<uint32_t>(__builtin_popcountll(mt & below)), in_round = 0;
    for (int w = 0; w < W; ++w) {
      const uint32_t c = sh.wave[buf][w][0];
      if (w < wave) pos += c;
      in_round += c;
    }
    if (in) emit(i, take, take ? pos : i - pos);
    round_end(base, taken0, in_round);
    taken0 += in_round;
  }
}

}  // namespace cfsel
