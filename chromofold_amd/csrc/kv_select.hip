// kv_select.hip — key bounds of page groups, selection of groups by a bound on their scores, eviction of groups by
// accumulated weight (chromofold/kv_select.h).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "cf_device.hpp"
#include "chromofold/kv_select.h"
#include "kv_topk.hpp"

namespace {

typedef int int4_t __attribute__((ext_vector_type(4)));
typedef float float4_t __attribute__((ext_vector_type(4)));

constexpr uint32_t kMaxGroups = 1u << 25;  // tables are shorter: 64 * max_groups fits 32 bits
constexpr int kRows = 16;                  // query heads of one KV head an MFMA tile takes

// Tokens of a sequence its query sees, and tokens its table can hold.
__device__ __forceinline__ uint32_t visible_tokens(uint32_t tokens, uint32_t pos, uint32_t max_groups) {
  if (tokens == 0) return 0;
  return min(min(tokens - 1, pos), 64 * max_groups - 1) + 1;  // (pos + 1 could wrap)
}

// ---- key bounds -------------------------------------------------------------------------------------------------
// One wavefront per group: a lane keeps 4 channels of every second (D = 128) or fourth (D = 64) token, 1 KiB per wavefront
// load. Max, min and a finiteness test of 4 D 64 B per group: bound by the read.
constexpr int kBoundWaves = 4;

template <int D>
__global__ __launch_bounds__(64 * kBoundWaves) void key_bounds_kernel(
    const float *__restrict__ keys, uint64_t ngroups, const uint64_t *__restrict__ first_page,
    const uint32_t *__restrict__ page_counts, const uint32_t *__restrict__ token_counts, const uint64_t *__restrict__ slots,
    int8_t *__restrict__ codes, float *__restrict__ scales, uint64_t slot_count) {
  constexpr int kL = D / 4;        // lanes of a token
  constexpr int kT = 64 / kL;      // tokens of a wavefront load
  constexpr int kIt = 16 / kT;     // loads of a page
  const int lane = threadIdx.x & 63;
  const uint64_t nw = static_cast<uint64_t>(gridDim.x) * kBoundWaves;
  for (uint64_t g = static_cast<uint64_t>(blockIdx.x) * kBoundWaves + (threadIdx.x >> 6); g < ngroups; g += nw) {
    const uint64_t slot = slots ? slots[g] : g;
    if (slot >= slot_count) continue;
    const uint32_t np = page_counts[g];
    const uint64_t p0 = first_page[g];
    float hi[4], lo[4], odd = 0.0f;  // odd: a NaN once a value was not finite
#pragma unroll
    for (int j = 0; j < 4; ++j) hi[j] = -INFINITY, lo[j] = -INFINITY;
    bool bad = np == 0 || np > CF_KV_GROUP_PAGES;
    uint32_t nt[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      nt[p] = bad || static_cast<uint32_t>(p) >= np ? 0u : token_counts ? token_counts[p0 + p] : 16u;
      bad |= !bad && static_cast<uint32_t>(p) < np && (nt[p] == 0 || nt[p] > 16u);
    }
    if (!bad) {
      float4_t x[4][kIt];  // the whole group in flight (absent pages: the last one again, no tokens of it)
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const float *page = keys + (p0 + min(static_cast<uint32_t>(p), np - 1)) * (16 * D);
#pragma unroll
        for (int i = 0; i < kIt; ++i)
          x[p][i] = __builtin_nontemporal_load(reinterpret_cast<const float4_t *>(page + (i * 64 + lane) * 4));
      }
      __builtin_amdgcn_sched_barrier(0);
      auto take = [&](auto masked) {
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
          for (int i = 0; i < kIt; ++i) {
            const bool here = !decltype(masked)::value || static_cast<uint32_t>(i * kT + lane / kL) < nt[p];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float v = x[p][i][j];
              hi[j] = fmaxf(hi[j], here ? v : -INFINITY);
              lo[j] = fmaxf(lo[j], here ? -v : -INFINITY);
              odd = __builtin_fmaf(here ? v : 0.0f, 0.0f, odd);
            }
          }
      };
      if ((nt[0] & nt[1] & nt[2] & nt[3]) == 16u) take(std::false_type{});
      else take(std::true_type{});
    }
#pragma unroll
    for (int o = kL; o < 64; o <<= 1)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        hi[j] = fmaxf(hi[j], __shfl_xor(hi[j], o));
        lo[j] = fmaxf(lo[j], __shfl_xor(lo[j], o));
      }
    bad |= __builtin_amdgcn_ballot_w64(odd != odd) != 0;
    float top = fmaxf(fmaxf(fmaxf(hi[0], lo[0]), fmaxf(hi[1], lo[1])), fmaxf(fmaxf(hi[2], lo[2]), fmaxf(hi[3], lo[3])));
#pragma unroll
    for (int o = 1; o < kL; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
    float s = bad ? INFINITY : top / 127.0f;
    // a subnormal quotient may have lost up to a third to rounding (all, from 0.5 steps down): up, so that 127 s is not below top
    if (s < 0x1p-126f && __builtin_fmaf(s, 127.0f, -top) < 0.0f) s = __uint_as_float(__float_as_uint(s) + 1);
    uint32_t ch = 0, cl = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      // outward, so that the codes bound the keys; |x| <= top: at most 127 but for the quotient's rounding
      const int a = bad ? 127 : s == 0.0f ? 0 : static_cast<int>(fmaxf(fminf(ceilf(hi[j] / s), 127.0f), -127.0f));
      const int b = bad ? 127 : s == 0.0f ? 0 : static_cast<int>(fmaxf(fminf(ceilf(lo[j] / s), 127.0f), -127.0f));
      ch |= (static_cast<uint32_t>(a) & 255u) << (8 * j);
      cl |= (static_cast<uint32_t>(b) & 255u) << (8 * j);
    }
    if (lane < kL) {
      uint32_t *rec = reinterpret_cast<uint32_t *>(codes + slot * (2 * D));
      rec[lane] = ch;
      rec[kL + lane] = cl;
      if (lane == 0) scales[slot] = s;
    }
  }
}

// ---- selection --------------------------------------------------------------------------------------------------
// Scores of 16 groups at a time on v_mfma_i32_16x16x64_i8: rows = the KV head's query heads, columns = groups, k = the 2 D
// products of one group, [max(a, 0), max(-a, 0)] . [upper codes, negated lower codes]. Whole numbers: a score does not depend
// on the order of its sum.
template <int D>
__device__ __forceinline__ void stage_query(const cf_kv_select_desc &d, uint32_t seq, uint32_t head, int8_t (*s_a)[2 * D],
                                            float *s_step, int nthreads) {
  const uint32_t gqa = d.query_head_count / d.kv_head_count;
  const int lane = threadIdx.x & 63;
  for (int h = threadIdx.x >> 6; h < kRows; h += nthreads >> 6) {  // a wavefront per query head
    constexpr int kN = D / 64;
    float q[kN], top = 0.0f;
    const float *row = d.queries + (static_cast<size_t>(seq) * d.query_head_count + head * gqa + h) * D;
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      q[j] = static_cast<uint32_t>(h) < gqa ? row[lane + 64 * j] : 0.0f;
      top = fmaxf(top, fabsf(q[j]));
    }
    top = cfd::rows4_max(cfd::row16_max(top));
    const float step = top / 127.0f;
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      const float r = q[j] / step;  // NaN for a NaN, for inf / inf and for 0 / 0: code 0
      const int a = r == r ? static_cast<int>(fmaxf(fminf(rintf(r), 127.0f), -127.0f)) : 0;
      s_a[h][lane + 64 * j] = static_cast<int8_t>(max(a, 0));
      s_a[h][D + lane + 64 * j] = static_cast<int8_t>(max(-a, 0));
    }
    if (lane == 0) s_step[h] = step;
  }
}

// Records of the 16 groups of a tile. Read as they lie, 1 KiB a wavefront load, and brought to the layout of a B operand
// (lane (kb, n): quarters of group n) through LDS: loads in that layout touch 64 lines each, at which one CU's cache gives
// 34 GB/s (a call of 8 rows of 2048 groups, one workgroup each, 22.7 us so, 16.5 through LDS).
template <int D>
struct Tile {
  static constexpr int kLoads = 2 * D / 64;
  static constexpr int kStride = 2 * D + 16;  // of a record in LDS: the 16 lanes of a read lie in different banks
  int4_t b[kLoads];
  float scale;  // of group n
  // ngroups: of the row that may be read
  __device__ __forceinline__ void load(const cf_kv_select_desc &d, size_t row, uint32_t tile, uint32_t ngroups) {
    constexpr int kL = 2 * D / 16;  // lanes of a record
    const int lane = threadIdx.x & 63;
    const int8_t *__restrict__ codes = d.codes + row * d.max_groups * (2 * D);
    const float *__restrict__ scales = d.scales + row * d.max_groups;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const size_t g = min(16 * tile + j * (64 / kL) + lane / kL, ngroups - 1);
      b[j] = *reinterpret_cast<const int4_t *>(codes + g * (2 * D) + 16 * (lane % kL));
    }
    scale = scales[min(16 * tile + (lane & 15), ngroups - 1)];
  }
  // Lane (kb, n) gets the products of group n with the heads 4 kb .. 4 kb + 3; lds: the wavefront's, 16 records.
  __device__ __forceinline__ int4_t products(const int4_t *a, int8_t *lds) const {
    constexpr int kL = 2 * D / 16;
    const int lane = threadIdx.x & 63, n = lane & 15, kb = lane >> 4;
#pragma unroll
    for (int j = 0; j < kLoads; ++j)
      *reinterpret_cast<int4_t *>(lds + (j * (64 / kL) + lane / kL) * kStride + 16 * (lane % kL)) = b[j];
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    int4_t c = {0, 0, 0, 0};
#pragma unroll
    for (int s = 0; s < kLoads; ++s)
      c = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[s], *reinterpret_cast<const int4_t *>(lds + n * kStride + 64 * s + 16 * kb), c,
                                                0, 0, 0);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    return c;
  }
};

// Keys (sortable scores) of a tile's units: lane n of the first sixteen has its group's (unit 1) or its pair's (unit 2) key,
// 0 where nothing is visible.
__device__ __forceinline__ uint32_t tile_keys(int4_t c, float scale, uint32_t tile, uint32_t ngroups, uint32_t unit, uint32_t gqa,
                                              const float *step) {
  const int lane = threadIdx.x & 63, n = lane & 15, kb = lane >> 4;
  float best = -INFINITY;  // a head whose step is not finite gives a NaN, which fmaxf passes over
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (static_cast<uint32_t>(4 * kb + r) < gqa) best = fmaxf(best, static_cast<float>(c[r]) * step[r]);
  best = cfd::rows4_max(best);
  uint32_t key = 16 * tile + n < ngroups ? cfsel::sortable(best * scale) : 0u;
  if (unit == 2) key = max(key, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(key), 0xb1, 0xf, 0xf, false)));
  return key;
}

template <int D>
struct QueryOperand {
  int4_t a[2 * D / 64];
  float step[4];
  __device__ __forceinline__ void load(const int8_t (*s_a)[2 * D], const float *s_step) {
    const int lane = threadIdx.x & 63, n = lane & 15, kb = lane >> 4;
#pragma unroll
    for (int s = 0; s < 2 * D / 64; ++s) a[s] = *reinterpret_cast<const int4_t *>(&s_a[n][64 * s + 16 * kb]);
#pragma unroll
    for (int r = 0; r < 4; ++r) step[r] = s_step[4 * kb + r];
  }
};

// Scores of the tiles wave0, wave0 + nwaves, ... of a row; put(unit, key) receives them. Two tiles at a time, the next
// ones' records loaded into their registers as soon as the products are formed (8 KiB a wavefront in flight at D = 128). The
// caller has loaded the first two, t, and staged the queries. All threads of the workgroup call this.
template <int D, typename Put>
__device__ __forceinline__ void score_row(const cf_kv_select_desc &d, size_t row, uint32_t ngroups, uint32_t wave0,
                                          uint32_t nwaves, Tile<D> (&t)[2], const int8_t (*s_a)[2 * D], const float *s_step,
                                          int8_t (*s_rec)[16 * Tile<D>::kStride], const Put &put) {
  const uint32_t tiles = (ngroups + 15) / 16, unit = d.unit_groups, gqa = d.query_head_count / d.kv_head_count;
  const int lane = threadIdx.x & 63;
  __syncthreads();
  QueryOperand<D> q;
  q.load(s_a, s_step);
  for (uint32_t i = wave0; i < tiles; i += 2 * nwaves) {
    int4_t c[2];
    float scale[2];
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j) {
      c[j] = t[j].products(q.a, s_rec[threadIdx.x >> 6]);
      scale[j] = t[j].scale;
      if (i + (j + 2) * nwaves < tiles) t[j].load(d, row, i + (j + 2) * nwaves, ngroups);
    }
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j) {
      const uint32_t tile = i + j * nwaves;
      if (tile >= tiles) break;
      const uint32_t key = tile_keys(c[j], scale[j], tile, ngroups, unit, gqa, q.step);
      if (lane < 16 && lane % unit == 0) put((16 * tile + lane) / unit, key);
    }
  }
}

__device__ __forceinline__ void fill_none(uint32_t *p, uint32_t from, uint32_t to, int nthreads) {
  for (uint32_t i = from + threadIdx.x; i < to; i += nthreads) p[i] = CF_KV_NO_UNIT;
}

template <int T, typename Keys>
__device__ __forceinline__ void pick_units(const cf_kv_select_desc &d, size_t row, uint32_t n, const Keys &keys,
                                           cfsel::TopkShared<T> &sh) {
  uint32_t *out = d.units + row * d.max_units;
  const uint32_t k = min(n, d.max_units);
  cfsel::take_largest<T>([&](uint32_t i) { return keys[i]; }, n, d.keep_first, d.keep_last, k, sh,
                         [&](uint32_t i, bool take, uint32_t pos) {
                           if (take) out[pos] = i;
                         },
                         [](uint32_t, uint32_t, uint32_t) {});
  fill_none(out, k, d.max_units, T);
}

__device__ __forceinline__ uint32_t visible_units(const cf_kv_select_desc &d, uint32_t ngroups) {
  return (ngroups + d.unit_groups - 1) / d.unit_groups;
}

// A row's scores and its best units in one workgroup of T threads, the keys in LDS: grid (KV heads, sequences).
constexpr uint32_t row_units_most(int T) { return T == 1024 ? 8192 : T == 512 ? 4096 : 2048; }

template <int D, int T>
__global__ __launch_bounds__(T) void select_row_kernel(cf_kv_select_desc d) {
  __shared__ __attribute__((aligned(16))) int8_t s_a[kRows][2 * D];
  __shared__ float s_step[kRows];
  __shared__ uint32_t s_key[row_units_most(T)];
  __shared__ __attribute__((aligned(16))) int8_t s_rec[T / 64][16 * Tile<D>::kStride];
  __shared__ cfsel::TopkShared<T> sh;
  const uint32_t head = blockIdx.x, seq = blockIdx.y;
  const uint32_t tokens = d.seq_tokens[seq], pos = d.query_pos[seq], wave = threadIdx.x >> 6;
  const size_t row = static_cast<size_t>(seq) * d.kv_head_count + head;
  // The first tiles and the queries do not wait for the row's length; what lies behind it is read for nothing (256 rows
  // x 512 groups 11.8 -> 11.0 us).
  Tile<D> t[2];
  t[0].load(d, row, wave, d.max_groups);
  stage_query<D>(d, seq, head, s_a, s_step, T);
  const uint32_t ngroups = (visible_tokens(tokens, pos, d.max_groups) + 63) / 64;
  const uint32_t n = visible_units(d, ngroups);
  if (n > d.max_units) {
    if (16 * (wave + T / 64) < ngroups) t[1].load(d, row, wave + T / 64, ngroups);
    score_row<D>(d, row, ngroups, wave, T / 64, t, s_a, s_step, s_rec, [&](uint32_t u, uint32_t key) {
      if (u < n) s_key[u] = key;
    });
    __syncthreads();
  }
  pick_units<T>(d, row, n, s_key, sh);
}

template <int D>
void launch_rows(const cf_kv_select_desc &d, int threads, hipStream_t s) {
  const dim3 grid(d.kv_head_count, d.seq_count);
  if (threads == 1024) select_row_kernel<D, 1024><<<grid, 1024, 0, s>>>(d);
  else if (threads == 512) select_row_kernel<D, 512><<<grid, 512, 0, s>>>(d);
  else select_row_kernel<D, 256><<<grid, 256, 0, s>>>(d);
}

// Two launches: scores to the workspace, grid (workgroups of a row, KV heads, sequences) ...
constexpr int kScoreThreads = 256;

template <int D>
__global__ __launch_bounds__(kScoreThreads) void score_kernel(cf_kv_select_desc d, uint32_t *__restrict__ keys,
                                                              uint32_t row_units) {
  __shared__ __attribute__((aligned(16))) int8_t s_a[kRows][2 * D];
  __shared__ float s_step[kRows];
  __shared__ __attribute__((aligned(16))) int8_t s_rec[kScoreThreads / 64][16 * Tile<D>::kStride];
  const uint32_t head = blockIdx.y, seq = blockIdx.z;
  const uint32_t ngroups = (visible_tokens(d.seq_tokens[seq], d.query_pos[seq], d.max_groups) + 63) / 64;
  constexpr uint32_t kPer = kScoreThreads / 64;
  if (16 * blockIdx.x * kPer >= ngroups) return;
  const size_t row = static_cast<size_t>(seq) * d.kv_head_count + head;
  uint32_t *out = keys + row * row_units;
  const uint32_t wave0 = blockIdx.x * kPer + (threadIdx.x >> 6), nwaves = gridDim.x * kPer;
  Tile<D> t[2];
#pragma unroll
  for (uint32_t j = 0; j < 2; ++j)
    if (16 * (wave0 + j * nwaves) < ngroups) t[j].load(d, row, wave0 + j * nwaves, ngroups);
  stage_query<D>(d, seq, head, s_a, s_step, kScoreThreads);
  score_row<D>(d, row, ngroups, wave0, nwaves, t, s_a, s_step, s_rec, [&](uint32_t u, uint32_t key) {
    if (u < row_units) out[u] = key;
  });
}

// ... and the best units of each row from there: grid (KV heads, sequences).
constexpr int kPickThreads = 1024;

__global__ __launch_bounds__(kPickThreads) void pick_kernel(cf_kv_select_desc d, const uint32_t *__restrict__ keys,
                                                            uint32_t row_units) {
  __shared__ cfsel::TopkShared<kPickThreads> sh;
  const uint32_t head = blockIdx.x, seq = blockIdx.y;
  const uint32_t ngroups = (visible_tokens(d.seq_tokens[seq], d.query_pos[seq], d.max_groups) + 63) / 64;
  const size_t row = static_cast<size_t>(seq) * d.kv_head_count + head;
  pick_units<kPickThreads>(d, row, visible_units(d, ngroups), keys + row * row_units, sh);
}

uint32_t row_units(const cf_kv_select_desc *d) { return (d->max_groups + d->unit_groups - 1) / d->unit_groups; }

// Threads of the one workgroup that takes a row, 0 for two launches (scores of a row over many workgroups, then the pick).
// us at 32 query / 8 KV heads, head_dim 128, as 256 / 512 / 1024 threads / two launches:
//   rows x groups   8 x 64     5.9 /  5.6 /  6.1 /  9.6     8 x 512  10.2 /  8.3 /  9.1 / 10.5     8 x 1024 15.0 / 10.8 / 10.9 / 10.8
//                   8 x 2048  24.2 / 16.4 / 15.1 / 11.9    32 x 2048 25.1 / 17.0 / 15.4 / 14.7    64 x 2048 27.6 / 18.0 / 15.7 / 17.7
//                 256 x 64     6.0 /  5.7 /  6.1 /  9.8   256 x 512  11.9 / 11.0 / 12.1 / 16.3   256 x 2048 33.1 / 26.1 / 25.7 / 31.0
//                 512 x 128    8.9 / 10.4 / 15.1 / 17.9   512 x 512  16.4 / 15.3 / 21.3 / 23.9   512 x 1024 27.1 / 25.4 / 29.1 / 34.8
//                1024 x 128   12.2 / 17.0 / 27.4 / 27.0  1024 x 256  15.8 / 18.5 / 33.5 / 30.2  1024 x 512  25.8 / 26.7 / 38.1 / 42.2
// Small workgroups leave several a CU, for more rows than CUs; a long row is read faster by many wavefronts, but one CU reads
// it at some 70 GB/s at best, which loses to two launches when other CUs would be idle.
int row_threads(const cf_kv_select_desc *d) {
  const uint32_t units = row_units(d);
  const bool many = static_cast<uint64_t>(d->seq_count) * d->kv_head_count > cfd::cu_count();
  const bool few = static_cast<uint64_t>(d->seq_count) * d->kv_head_count < 64;
  const uint64_t row_bytes = static_cast<uint64_t>(d->max_groups) * 2 * d->head_dim;
  if (units > row_units_most(1024) || (few && row_bytes > (256u << 10))) return 0;
  if (many && d->max_groups <= 256) return 256;
  return units <= row_units_most(512) && (many || d->max_groups <= 1024) ? 512 : 1024;
}

// ---- eviction ---------------------------------------------------------------------------------------------------
struct Budget {
  uint32_t tokens, groups, units, kept;
  __device__ Budget(const cf_kv_evict_desc &d, uint32_t t) {
    tokens = min(t, 64 * d.max_groups);
    groups = tokens / 64 + (tokens % 64 != 0);
    units = groups / d.unit_groups + (groups % d.unit_groups != 0);
    kept = min(units, d.budget_units);
  }
  __device__ uint32_t tokens_out(const cf_kv_evict_desc &d) const { return tokens - 64 * d.unit_groups * (units - kept); }
};

__global__ void evict_tokens_kernel(cf_kv_evict_desc d) {
  const uint32_t s = blockIdx.x * blockDim.x + threadIdx.x;
  if (s < d.seq_count) d.seq_tokens_out[s] = Budget(d, d.seq_tokens[s]).tokens_out(d);
}

constexpr uint32_t kEvictKeys = 8192;  // keys of a row that are held in LDS; longer rows read their weights again

// Workgroups of T threads, grid (KV heads, sequences, parts of a row; one in place). Units are decided and moved in rounds of T of them in index order: a
// kept unit moves down or stays, so a round's destinations lie at or before its sources and before every later round's;
// within a step all reads come before the first write. That is what makes eviction in place safe. Bound by latency: the
// weights, the pick, then one read and one write of everything a step moves.
template <int D, int T>
__global__ __launch_bounds__(T) void evict_kernel(cf_kv_evict_desc d, bool tokens_here) {
  constexpr uint32_t kL = 2 * D / 16;       // 16-byte pieces of a record
  constexpr uint32_t kPer = 8;              // pieces a thread moves in a step
  constexpr uint32_t kStep = T * kPer / kL; // groups of a step
  __shared__ cfsel::TopkShared<T> sh;
  __shared__ uint32_t s_from[2 * T];  // source groups of the round's kept groups
  __shared__ uint32_t s_key[kEvictKeys];
  const uint32_t head = blockIdx.x, seq = blockIdx.y, part = blockIdx.z, parts = gridDim.z, unit = d.unit_groups;
  const uint32_t tid = threadIdx.x;
  const Budget b(d, d.seq_tokens[seq]);
  const size_t row = (static_cast<size_t>(seq) * d.kv_head_count + head) * d.max_groups;
  const float *w = d.weights + row;
  const uint32_t *off = d.group_offsets + row;
  auto key_of = [&](uint32_t u) {
    float x = w[u * unit];
    if (unit == 2 && 2 * u + 1 < b.groups) x += w[2 * u + 1];
    return cfsel::sortable(x);
  };
  const bool held = b.units <= kEvictKeys;
  if (held && b.units > b.kept) {
    for (uint32_t u = tid; u < b.units; u += T) s_key[u] = key_of(u);
    __syncthreads();
  }
  cfsel::take_largest<T>(
      [&](uint32_t u) { return held ? s_key[u] : key_of(u); }, b.units, d.keep_first, d.keep_last, b.kept, sh,
      [&](uint32_t u, bool take, uint32_t pos) {
        for (uint32_t j = 0; j < unit; ++j) {
          const uint32_t g = u * unit + j;
          if (take) {
            if (g < b.groups) s_from[(pos * unit + j) % (2 * T)] = g;
          } else if (d.dropped && part == 0) {
            d.dropped[row + pos * unit + j] = off[g];  // a dropped unit is not the last: all its groups exist
          }
        }
      },
      [&](uint32_t, uint32_t before, uint32_t cnt) {
        // kept groups of the round, [g0, g1) of them this part's; s_from is read at the same positions modulo its size
        const uint32_t most = b.groups - (b.units - b.kept) * unit;
        const uint32_t r0 = min(before * unit, most), r1 = min((before + cnt) * unit, most);
        const uint32_t share = (r1 - r0 + parts - 1) / parts;
        const uint32_t g0 = min(r0 + part * share, r1), g1 = min(g0 + share, r1);
        __syncthreads();
        for (uint32_t a = g0; a < g1; a += kStep) {
          const uint32_t i = a + tid, m = min(g1 - a, kStep) * kL;
          const bool in = tid < kStep && i < g1;
          uint32_t o = 0;
          float x = 0.0f, sc = 0.0f;
          int4_t v[kPer];
          if (in) {
            const uint32_t src = s_from[i % (2 * T)];
            o = off[src];
            if (d.weights_out) x = w[src];
            if (d.codes_out) sc = d.scales[row + src];
          }
          if (d.codes_out) {
#pragma unroll
            for (uint32_t e = 0; e < kPer; ++e) {
              const uint32_t p = e * T + tid;
              if (p < m)
                v[e] = *reinterpret_cast<const int4_t *>(d.codes + (row + s_from[(a + p / kL) % (2 * T)]) * (2 * D) +
                                                         16 * (p % kL));
            }
          }
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // every read of this wavefront has returned
          __syncthreads();
          if (in) {
            d.group_offsets_out[row + i] = o;
            if (d.weights_out) d.weights_out[row + i] = x;
            if (d.codes_out) d.scales_out[row + i] = sc;
          }
          if (d.codes_out) {
#pragma unroll
            for (uint32_t e = 0; e < kPer; ++e) {
              const uint32_t p = e * T + tid;
              if (p < m) *reinterpret_cast<int4_t *>(d.codes_out + (row + a + p / kL) * (2 * D) + 16 * (p % kL)) = v[e];
            }
          }
        }
        __syncthreads();  // s_from is free for the next round
      });
  const uint32_t left = b.groups - (b.units - b.kept) * unit, gone = b.groups - left;
  __syncthreads();  // every weight has been read
  if (part != 0) return;
  if (d.weights_out)
    for (uint32_t i = left + tid; i < d.max_groups; i += T) d.weights_out[row + i] = 0.0f;
  if (d.dropped)
    for (uint32_t i = gone + tid; i < d.max_groups; i += T) d.dropped[row + i] = CF_KV_NO_UNIT;
  if (tokens_here && head == 0 && tid == 0) d.seq_tokens_out[seq] = b.tokens_out(d);
}

// Workgroups of a row: each picks all of it and moves its part of what stays, where no array is written that they read and
// CUs would be idle (one of 1024 threads fits a CU). us, of 1024 threads, with 1 / 2 / 4 / 8 / 16 of them: 32 rows, 1024 of 2048 groups
// 15.1 / 12.4 / 11.3 / 10.9 / 17.9; 8 rows, 64 of 128 groups 6.3 / 6.0 / 5.8 / 5.8 / 5.8, 4000 of 7813 groups
// 49.6 / 38.2 / 34.2 / 32.2 / 30.8; 256 rows, 256 of 512 groups 13.2 / 21.1 / 35.5.
uint32_t evict_parts(const cf_kv_evict_desc &d) {
  const bool apart = d.group_offsets_out != d.group_offsets && d.weights_out != d.weights &&
                     (!d.codes_out || (d.codes_out != d.codes && d.scales_out != d.scales));
  const uint64_t rows = static_cast<uint64_t>(d.seq_count) * d.kv_head_count;
  return apart ? static_cast<uint32_t>(std::clamp<uint64_t>(cfd::cu_count() / rows, 1, 16)) : 1u;
}

template <int D>
void launch_evict(const cf_kv_evict_desc &d, bool tokens_here, hipStream_t s) {
  const dim3 grid(d.kv_head_count, d.seq_count, evict_parts(d));
  // us with 256 / 512 / 1024 threads: 8 rows, 64 of 128 groups 5.7 / 6.1 / 7.2, 256 rows, 128 of 256 8.9 / 8.7 / 9.5, 256
  // of 512 14.0 / 12.4 / 13.5, 512 of 1024 22.5 / 20.1 / 18.9; 512 rows, 512 of 1024 37.9 / 34.4 / 41.0
  const uint32_t units = (d.max_groups + d.unit_groups - 1) / d.unit_groups;
  const bool many = static_cast<uint64_t>(d.seq_count) * d.kv_head_count > cfd::cu_count();
  if (units <= 256) evict_kernel<D, 256><<<grid, 256, 0, s>>>(d, tokens_here);
  else if (units <= 512 || many) evict_kernel<D, 512><<<grid, 512, 0, s>>>(d, tokens_here);
  else evict_kernel<D, 1024><<<grid, 1024, 0, s>>>(d, tokens_here);
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
// grids have the sequences or KV heads in y and z
bool shape_ok(uint32_t seqs, uint32_t heads) { return seqs <= 65535 && heads <= 65535; }

}  // namespace

extern "C" cf_status cf_kv_key_bounds_async(const float *keys, uint64_t ngroups, const uint64_t *first_page,
                                            const uint32_t *page_counts, const uint32_t *token_counts, uint32_t head_dim,
                                            const uint64_t *slots, int8_t *codes, float *scales, uint64_t slot_count,
                                            void *stream) {
  if (!keys || !first_page || !page_counts || !codes || !scales || ngroups == 0) return CF_ERR_INVALID_ARGUMENT;
  if (!aligned16(keys) || !aligned16(codes)) return CF_ERR_INVALID_ARGUMENT;
  if (head_dim != 64 && head_dim != 128) return CF_ERR_UNSUPPORTED;
  const uint64_t wg = (ngroups + kBoundWaves - 1) / kBoundWaves;
  const dim3 grid(static_cast<uint32_t>(std::min<uint64_t>(wg, 1u << 20)));
  const hipStream_t s = cfd::as_stream(stream);
  if (head_dim == 128)
    key_bounds_kernel<128><<<grid, 64 * kBoundWaves, 0, s>>>(keys, ngroups, first_page, page_counts, token_counts, slots,
                                                             codes, scales, slot_count);
  else
    key_bounds_kernel<64><<<grid, 64 * kBoundWaves, 0, s>>>(keys, ngroups, first_page, page_counts, token_counts, slots,
                                                            codes, scales, slot_count);
  return cfd::launch_status();
}

extern "C" cf_status cf_kv_validate_select_desc(const cf_kv_select_desc *d) {
  if (!d || d->struct_size != sizeof(cf_kv_select_desc) || d->abi_version != CF_KV_SELECT_ABI_VERSION)
    return CF_ERR_INVALID_ARGUMENT;
  if (!d->codes || !d->scales || !d->seq_tokens || !d->query_pos || !d->queries || !d->units || d->seq_count == 0 ||
      d->kv_head_count == 0 || d->query_head_count == 0 || d->query_head_count % d->kv_head_count != 0 ||
      d->max_groups == 0 || d->max_units == 0 || !aligned16(d->codes))
    return CF_ERR_INVALID_ARGUMENT;
  if (d->unit_groups != 1 && d->unit_groups != 2) return CF_ERR_INVALID_ARGUMENT;
  if (d->keep_first > d->max_units || d->keep_last > d->max_units - d->keep_first) return CF_ERR_INVALID_ARGUMENT;
  if (d->head_dim != 64 && d->head_dim != 128) return CF_ERR_UNSUPPORTED;
  if (d->query_head_count / d->kv_head_count > CF_KV_SELECT_MAX_GQA) return CF_ERR_UNSUPPORTED;
  if (!shape_ok(d->seq_count, d->kv_head_count) || d->max_groups >= kMaxGroups) return CF_ERR_UNSUPPORTED;
  return CF_OK;
}

extern "C" uint64_t cf_kv_select_workspace_bytes(const cf_kv_select_desc *d) {
  if (cf_kv_validate_select_desc(d) != CF_OK || row_threads(d)) return 0;
  return static_cast<uint64_t>(d->seq_count) * d->kv_head_count * row_units(d) * sizeof(uint32_t);
}

extern "C" cf_status cf_kv_select_groups_async(const cf_kv_select_desc *d, void *stream) {
  const cf_status v = cf_kv_validate_select_desc(d);
  if (v != CF_OK) return v;
  const uint64_t need = cf_kv_select_workspace_bytes(d);
  if (need && (!d->workspace || d->workspace_bytes < need || !aligned16(d->workspace))) return CF_ERR_INVALID_ARGUMENT;
  const hipStream_t s = cfd::as_stream(stream);
  if (const int threads = row_threads(d)) {
    if (d->head_dim == 128) launch_rows<128>(*d, threads, s);
    else launch_rows<64>(*d, threads, s);
    return cfd::launch_status();
  }
  const uint32_t units = row_units(d);
  uint32_t *keys = static_cast<uint32_t *>(d->workspace);
  const uint32_t tiles = (d->max_groups + 15) / 16, per = kScoreThreads / 64;
  // wavefronts of about 4 tiles where there are enough rows to fill the chip with them
  const uint64_t rows = static_cast<uint64_t>(d->kv_head_count) * d->seq_count;
  const uint32_t most = std::max<uint32_t>((tiles + per - 1) / per, 1u);
  const uint64_t want = std::max<uint64_t>((most + 3) / 4, (4ull * cfd::cu_count() + rows - 1) / rows);
  const dim3 grid(static_cast<uint32_t>(std::min<uint64_t>({want, most, 1u << 16})), d->kv_head_count, d->seq_count);
  if (d->head_dim == 128) score_kernel<128><<<grid, kScoreThreads, 0, s>>>(*d, keys, units);
  else score_kernel<64><<<grid, kScoreThreads, 0, s>>>(*d, keys, units);
  pick_kernel<<<dim3(d->kv_head_count, d->seq_count), kPickThreads, 0, s>>>(*d, keys, units);
  return cfd::launch_status();
}

extern "C" cf_status cf_kv_validate_evict_desc(const cf_kv_evict_desc *d) {
  if (!d || d->struct_size != sizeof(cf_kv_evict_desc) || d->abi_version != CF_KV_SELECT_ABI_VERSION)
    return CF_ERR_INVALID_ARGUMENT;
  if (!d->group_offsets || !d->seq_tokens || !d->weights || !d->group_offsets_out || !d->seq_tokens_out ||
      d->seq_count == 0 || d->kv_head_count == 0 || d->max_groups == 0 || d->budget_units == 0)
    return CF_ERR_INVALID_ARGUMENT;
  if (d->unit_groups != 1 && d->unit_groups != 2) return CF_ERR_INVALID_ARGUMENT;
  if (d->keep_last == 0 || d->keep_first > d->budget_units || d->keep_last > d->budget_units - d->keep_first)
    return CF_ERR_INVALID_ARGUMENT;
  const int records = (d->codes != nullptr) + (d->scales != nullptr) + (d->codes_out != nullptr) + (d->scales_out != nullptr);
  if ((records != 0 && records != 4) || !aligned16(d->codes) || !aligned16(d->codes_out)) return CF_ERR_INVALID_ARGUMENT;
  if (d->head_dim != 64 && d->head_dim != 128) return CF_ERR_UNSUPPORTED;
  if (!shape_ok(d->seq_count, d->kv_head_count) || d->max_groups >= kMaxGroups) return CF_ERR_UNSUPPORTED;
  return CF_OK;
}

extern "C" cf_status cf_kv_evict_groups_async(const cf_kv_evict_desc *d, void *stream) {
  const cf_status v = cf_kv_validate_evict_desc(d);
  if (v != CF_OK) return v;
  const hipStream_t s = cfd::as_stream(stream);
  // in place, the lengths are still read by the workgroups of the other heads: a launch of their own behind them
  const bool tokens_here = d->seq_tokens_out != d->seq_tokens;
  if (d->head_dim == 128) launch_evict<128>(*d, tokens_here, s);
  else launch_evict<64>(*d, tokens_here, s);
  if (!tokens_here) evict_tokens_kernel<<<cfd::grid_for(d->seq_count, 256), 256, 0, s>>>(*d);
  return cfd::launch_status();
}
