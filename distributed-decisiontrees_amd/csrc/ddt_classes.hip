// ddt_classes.hip -- operators on a matrix of class scores (row r, class c): adjust (penalties for repeated classes, biases, masks),
// top (the k best classes of each row and the row's log-sum-exp), distill (a student's loss against a teacher's top scores, and its
// gradient).  All of them read the matrix once from HBM and do little per score: bandwidth is what bounds them.
//
// A 16-byte piece of a row is a "pack" (4 fp32 or 8 two-byte scores).  Rows start at any address (an odd number of classes): global
// memory takes a 16-byte access at any element address, so packs count from the row's own start and only a row's last pack is partial.
// Arithmetic is fp32 or wider whatever the scores' type; a result is rounded once, to nearest even, when it is stored.
#include <hip/hip_runtime.h>
#include <float.h>
#include <math.h>

#include <type_traits>

#include "../../include/ddt.h"
#include "ddt_classes.h"

namespace ddt {
namespace {

extern __shared__ uint32_t lds_words[];

constexpr float kInf = __builtin_inff();

template <class T>
struct Pack {
  static constexpr uint32_t N = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(16 / sizeof(T))));
};

// scores [c, c + N) of a row of `end` classes; `fill` behind its end
template <class T>
__device__ __forceinline__ void load_pack(const T* row, uint32_t c, uint32_t end, float fill, float (&x)[Pack<T>::N]) {
  constexpr uint32_t N = Pack<T>::N;
  if (c + N <= end) {
    typename Pack<T>::vec v;
    __builtin_memcpy(&v, row + c, 16);
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) x[i] = (float)v[i];
  } else {
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) x[i] = c + i < end ? (float)row[c + i] : fill;
  }
}
// four packs, STEP packs apart, some of them partial or behind the end: `fill` there
template <class T, uint32_t STEP>
__device__ __forceinline__ void load_last_packs(const T* row, uint32_t p, uint32_t end, float fill, float (&x)[4 * Pack<T>::N]) {
  constexpr uint32_t N = Pack<T>::N;
#pragma unroll
  for (uint32_t u = 0; u < 4; ++u) {
    float v[N];
    load_pack(row, (p + u * STEP) * N, end, fill, v);
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) x[u * N + i] = v[i];
  }
}
// four whole packs, STEP packs apart
template <class T, uint32_t STEP>
__device__ __forceinline__ void load_packs(const T* row, uint32_t p, float (&x)[4 * Pack<T>::N]) {
  constexpr uint32_t N = Pack<T>::N;
  typename Pack<T>::vec v[4];
#pragma unroll
  for (uint32_t u = 0; u < 4; ++u) __builtin_memcpy(&v[u], row + (size_t)(p + u * STEP) * N, 16);
#pragma unroll
  for (uint32_t u = 0; u < 4; ++u)
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) x[u * N + i] = (float)v[u][i];
}
// PAST: nontemporal, so that what is written does not push out what will be read again
template <class T, bool PAST = false>
__device__ __forceinline__ void store_pack(T* row, uint32_t c, uint32_t end, const float (&x)[Pack<T>::N]) {
  constexpr uint32_t N = Pack<T>::N;
  if (c + N <= end) {
    typename Pack<T>::vec v;
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) v[i] = (T)x[i];
    typedef typename Pack<T>::vec anywhere __attribute__((aligned(sizeof(T))));
    if (PAST) __builtin_nontemporal_store(v, reinterpret_cast<anywhere*>(row + c));
    else __builtin_memcpy(row + c, &v, 16);
  } else {
#pragma unroll
    for (uint32_t i = 0; i < N; ++i)
      if (c + i < end) row[c + i] = (T)x[i];
  }
}

// A pack kept in registers as it came.  hold() ends what the compiler may carry over from one use to the next: without it the fp32
// forms of all packs stay live beside the packs themselves, twice the registers.
template <class T>
struct HeldPack {
  static constexpr uint32_t N = Pack<T>::N;
  uint32_t w[4];
  __device__ __forceinline__ void load(const T* row, uint32_t c, uint32_t end) {
    if (c + N <= end) {
      __builtin_memcpy(w, row + c, 16);
    } else {
      typename Pack<T>::vec v;
#pragma unroll
      for (uint32_t i = 0; i < N; ++i) v[i] = c + i < end ? row[c + i] : (T)-kInf;
      __builtin_memcpy(w, &v, 16);
    }
  }
  __device__ __forceinline__ void get(float (&x)[N]) const {
    typename Pack<T>::vec v;
    __builtin_memcpy(&v, w, 16);
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) x[i] = (float)v[i];
  }
  __device__ __forceinline__ void clear(uint32_t bits) {  // -inf where a bit is set
    typename Pack<T>::vec v;
    __builtin_memcpy(&v, w, 16);
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) v[i] = (bits >> i) & 1u ? (T)-kInf : v[i];
    __builtin_memcpy(w, &v, 16);
  }
  __device__ __forceinline__ void hold() { asm volatile("" : "+v"(w[0]), "+v"(w[1]), "+v"(w[2]), "+v"(w[3])); }
};

// What is computed from a thread's number is the same for every row, and the compiler keeps all of it across the loop over rows: twice the
// registers for nothing (most blocks take one row).  forget() makes the number new to it.
__device__ __forceinline__ void forget(uint32_t& v) { asm volatile("" : "+v"(v)); }
__device__ __forceinline__ uint32_t forgotten(uint32_t v) {
  forget(v);
  return v;
}

// 2 ^ x: the hardware instruction (1 ulp; results below 2^-126 may come back as 0 -- nothing next to a sum whose largest term is 1)
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// 2^y and ln v beyond fp32 for the rows' own numbers.  2^y: y = n + f with |f| <= 1/2, the power series of e^(f ln 2) to the 10th power in
// 64 bits (the 11th is below 3e-13 of the sum; a loss is a difference of such logarithms, and where a student has learned its teacher
// one of 1e-4 is left of terms near 10: 3e-8 of it), scaled by 2^n: a third of the instructions of the library's exp, which aims at the
// last of the 64 bits.
__device__ __forceinline__ double exp2_64(double y) {
  y = y < -1100.0 ? -1100.0 : y > 1100.0 ? 1100.0 : y;  // (NaN stays)
  const double n = __builtin_rint(y), f = (y - n) * 0.69314718055994530942;
  double p = 1.0 / 3628800.0;
  p = fma(p, f, 1.0 / 362880.0);
  p = fma(p, f, 1.0 / 40320.0);
  p = fma(p, f, 1.0 / 5040.0);
  p = fma(p, f, 1.0 / 720.0);
  p = fma(p, f, 1.0 / 120.0);
  p = fma(p, f, 1.0 / 24.0);
  p = fma(p, f, 1.0 / 6.0);
  p = fma(p, f, 0.5);
  p = fma(p, f, 1.0);
  p = fma(p, f, 1.0);
  return __builtin_amdgcn_ldexp(p, (int)n);
}
// ln v: the fp32 logarithm and one Newton step on 2^y = v.  For 0 and the normal fp32 range, which sums relative to their largest term
// and probabilities that count stay in.
__device__ __forceinline__ double log_64(double v) {
  if (v == 0.0) return -__builtin_inf();
  const double y = (double)__builtin_amdgcn_logf((float)v), r = fma(v, exp2_64(-y), -1.0);
  return fma(y, 0.69314718055994530942, r - 0.5 * r * r);
}

// 1 / v for sums relative to their largest term: the hardware's first digits and two Newton steps
__device__ __forceinline__ double inverse_64(double v) {
  double r = __builtin_amdgcn_rcp(v);
  r = fma(fma(-v, r, 1.0), r, r);
  return fma(fma(-v, r, 1.0), r, r);
}

// reductions over a wave: five moves within rows of 16 lanes and across them (DPP: no LDS), the last lane then holds the result of all
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp(float idle, float v) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp((int)__float_as_uint(idle), (int)__float_as_uint(v), CTRL, ROWS, 0xF, false));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp(uint32_t idle, uint32_t v) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)idle, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp(double idle, double v) {
  const uint64_t i = (uint64_t)__double_as_longlong(idle), b = (uint64_t)__double_as_longlong(v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp((int)(uint32_t)i, (int)(uint32_t)b, CTRL, ROWS, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp((int)(uint32_t)(i >> 32), (int)(uint32_t)(b >> 32), CTRL, ROWS, 0xF, false);
  return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
constexpr int kRowShr1 = 0x111, kRowShr2 = 0x112, kRowShr4 = 0x114, kRowShr8 = 0x118, kRowBcast15 = 0x142, kRowBcast31 = 0x143;
__device__ __forceinline__ float last_lane(float v) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), 63)); }
__device__ __forceinline__ double last_lane(double v) {
  const uint64_t b = (uint64_t)__double_as_longlong(v);
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)b, 63), hi = __builtin_amdgcn_readlane((uint32_t)(b >> 32), 63);
  return __longlong_as_double((long long)((uint64_t)hi << 32 | lo));
}
template <class F>
__device__ __forceinline__ F wave_sum(F v) {
  v += dpp<kRowShr1, 0xF>((F)0, v);
  v += dpp<kRowShr2, 0xF>((F)0, v);
  v += dpp<kRowShr4, 0xF>((F)0, v);
  v += dpp<kRowShr8, 0xF>((F)0, v);
  v += dpp<kRowBcast15, 0xA>((F)0, v);
  v += dpp<kRowBcast31, 0xC>((F)0, v);
  return last_lane(v);
}
// ... and over NT lanes of a row of scores: 16 (rotations within the row of lanes, every lane holds the result) or the whole wave
constexpr int kRowRor1 = 0x121, kRowRor2 = 0x122, kRowRor4 = 0x124, kRowRor8 = 0x128;
__device__ __forceinline__ float wave_max(float v) {
  v = fmaxf(v, dpp<kRowShr1, 0xF>(v, v));
  v = fmaxf(v, dpp<kRowShr2, 0xF>(v, v));
  v = fmaxf(v, dpp<kRowShr4, 0xF>(v, v));
  v = fmaxf(v, dpp<kRowShr8, 0xF>(v, v));
  v = fmaxf(v, dpp<kRowBcast15, 0xA>(v, v));
  v = fmaxf(v, dpp<kRowBcast31, 0xC>(v, v));
  return last_lane(v);
}

template <int NT, class F>
__device__ __forceinline__ F lanes_sum(F v) {
  if (NT != 16) return wave_sum(v);
  v += dpp<kRowRor8, 0xF>((F)0, v);
  v += dpp<kRowRor4, 0xF>((F)0, v);
  v += dpp<kRowRor2, 0xF>((F)0, v);
  v += dpp<kRowRor1, 0xF>((F)0, v);
  return v;
}
template <int NT>
__device__ __forceinline__ float lanes_max(float v) {
  if (NT != 16) return wave_max(v);
  v = fmaxf(v, dpp<kRowRor8, 0xF>(v, v));
  v = fmaxf(v, dpp<kRowRor4, 0xF>(v, v));
  v = fmaxf(v, dpp<kRowRor2, 0xF>(v, v));
  v = fmaxf(v, dpp<kRowRor1, 0xF>(v, v));
  return v;
}

// ---------------------------------------------------------------------------------------------------
// adjust
// ---------------------------------------------------------------------------------------------------
// word of the history counter: times the class stands behind the row's prompt part, bit 31 = it stands in the prompt part
constexpr uint32_t kInPrompt = 0x80000000u;

struct RowPenalty {
  float rep, freq, pres;
};
__device__ __forceinline__ RowPenalty row_penalty(const AdjustArgs& a, uint64_t r) {
  return {a.repetition ? a.repetition[r] : 1.f, a.frequency ? a.frequency[r] : 0.f, a.presence ? a.presence[r] : 0.f};
}
__device__ __forceinline__ float penalise(float x, uint32_t w, const RowPenalty& p) {
  if (w == 0u) return x;
  x = x > 0.f ? x / p.rep : x * p.rep;
  const uint32_t behind = w & ~kInPrompt;
  x = x - p.freq * (float)behind;
  return behind ? x - p.pres : x;
}

// zeroes `words` counters (rounded up to 4) and counts the history of rows [r0, r0 + rows) for classes [c0, c0 + C) into
// counts[r * row_pitch + c * class_pitch].  Integer LDS adds: their order does not show.  Offsets and class numbers come from the device
// unchecked: offsets are clamped to the history's length, numbers outside the tile (also outside the matrix) count nowhere.
template <uint32_t kAhead>
__device__ __forceinline__ void count_history(const AdjustArgs& a, uint64_t r0, uint32_t rows, uint32_t c0, uint32_t C, uint32_t row_pitch,
                                              uint32_t class_pitch, uint32_t words, uint32_t* counts) {
  const uint32_t waves = blockDim.x >> 6;
  const bool per_wave = rows >= waves;  // a wave per row; fewer rows than waves: all threads on one row after the other
  const uint32_t step = (per_wave ? 64u : blockDim.x) * 4u, start = (per_wave ? threadIdx.x & 63u : threadIdx.x) * 4u;
  uint32_t r = per_wave ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0u;
  int64_t lo, split, hi;
  auto offsets = [&] {
    const int64_t len = (int64_t)a.history_len;
    lo = a.first[r0 + r], hi = a.first[r0 + r + 1], split = a.prompt ? (int64_t)a.prompt[r0 + r] : 0;
    lo = lo < 0 ? 0 : lo > len ? len : lo;
    hi = hi < lo ? lo : hi > len ? len : hi;
    split = split < 0 ? lo : split > hi - lo ? hi : lo + split;
  };
  offsets();  // (r < rows) under way while the counters are cleared
  __syncthreads();  // the tile before has been read
  for (uint32_t i = threadIdx.x; i < (words + 3u) / 4u; i += blockDim.x) reinterpret_cast<uint4*>(counts)[i] = make_uint4(0u, 0u, 0u, 0u);
  __syncthreads();
  while (r < rows) {
    uint32_t* row = counts + r * row_pitch;
    // kAhead 16-byte loads of a thread in flight: every tile of the row reads the whole history (from L2), and one entry at a time
    // that is 400 dependent loads for 100,000 entries.  Four for the long histories of 1024 threads (50,000 entries a row 21.7 -> 20.8 us),
    // two elsewhere (four: 4096 entries a row 19.1 -> 19.9 us, 64 entries 43 -> 49)
    auto count_part = [&](int64_t from, int64_t to, bool in_prompt) {
      for (; from < to; from += 1 << 30) {  // (32-bit positions inside a piece)
        const int32_t* h = a.history + from;
        const uint32_t n = (uint32_t)(to - from < (1 << 30) ? to - from : (1 << 30));
        for (uint32_t i = start; i < n; i += step * kAhead) {
          uint32_t c[kAhead][4];
#pragma unroll
          for (uint32_t u = 0; u < kAhead; ++u) {
            const uint32_t at = i + u * step;
            if (at + 4u <= n) __builtin_memcpy(c[u], h + at, 16);
            else {
#pragma unroll
              for (uint32_t j = 0; j < 4; ++j) c[u][j] = at + j < n ? (uint32_t)h[at + j] : 0xFFFFFFFFu;
            }
          }
#pragma unroll
          for (uint32_t u = 0; u < kAhead; ++u)
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)
              if (c[u][j] - c0 < C) {
                if (in_prompt) atomicOr(&row[(c[u][j] - c0) * class_pitch], kInPrompt);
                else atomicAdd(&row[(c[u][j] - c0) * class_pitch], 1u);
              }
        }
      }
    };
    count_part(lo, split, true);
    count_part(split, hi, false);
    r += per_wave ? waves : 1u;
    if (r < rows) offsets();
  }
  __syncthreads();
}

struct AdjustTiles {
  uint32_t rows, classes;      // of a tile; row-major: classes is a multiple of the pack
  uint32_t magic;              // row-major: idx / (classes / N) = umulhi(idx, magic)
  uint64_t class_tiles, tiles;
};

// Row-major: a tile is `rows` rows times `classes` classes, at most NT * ITER packs of them, ITER per thread.  All loads of a thread --
// scores, bias, mask, the row's penalties -- are on their way before the history is counted.  What bounds it with a history is the chain of
// a tile's latencies (offsets, entries, counters, scores): 64 x 128000 bf16 takes 10 us without histories, 14 with 10 entries a row, 18 with
// 4096; 32 x 50257 fp32 with 50,000 entries a row 20 us, six rounds of loads for the longest row.  A row's tiles lie on all eight XCDs, and
// each of their L2s fetches the history for itself: 61 MB where scores and histories once are 13, 26 where they are 18.5.
template <class T, bool HIST, int NT, int ITER>
__global__ __launch_bounds__(NT) void adjust_rows_kernel(const AdjustArgs a, const AdjustTiles t) {
  constexpr uint32_t N = Pack<T>::N;
  const uint32_t ppr = t.classes / N;
  for (uint64_t tile = blockIdx.x; tile < t.tiles; tile += gridDim.x) {
    const uint64_t rt = tile / t.class_tiles, r0 = rt * t.rows;
    const uint32_t c0 = (uint32_t)(tile - rt * t.class_tiles) * t.classes;
    const uint32_t rows = (uint32_t)(a.n - r0 < t.rows ? a.n - r0 : t.rows);
    const uint32_t C = a.K - c0 < t.classes ? a.K - c0 : t.classes;
    const uint32_t tid = forgotten(threadIdx.x);
    HeldPack<T> raw[ITER];
    float bias[ITER][N];
    uint32_t bits[ITER], q[ITER], cl[ITER];
    RowPenalty pen[ITER];
#pragma unroll
    for (int u = 0; u < ITER; ++u) {
      const uint32_t idx = tid + (uint32_t)u * NT;
      q[u] = t.rows == 1u ? 0u : ppr == 1u ? idx : __umulhi(idx, t.magic), cl[u] = (idx - q[u] * ppr) * N;
      const uint32_t c = c0 + cl[u];
      const uint64_t r = r0 + q[u];
      bits[u] = 0xFFFFFFFFu;
#pragma unroll
      for (uint32_t i = 0; i < N; ++i) bias[u][i] = 0.f;
      if (q[u] >= rows || cl[u] >= C) continue;
      raw[u].load(static_cast<const T*>(a.in) + r * a.in_stride, c, a.K);
      if (a.allowed) bits[u] = a.allowed[r * a.allowed_rs + (c >> 5)] >> (c & 31u);  // (a pack's bits stand in one word)
      if (HIST) pen[u] = row_penalty(a, r);
      if (a.bias) {
        const float* b = a.bias + r * a.bias_rs;
        if (a.bias_cs == 1u && c + N <= a.K) {
          __builtin_memcpy(bias[u], b + c, sizeof(bias[u]));
        } else {
#pragma unroll
          for (uint32_t i = 0; i < N; ++i)
            if (c + i < a.K) bias[u][i] = b[(uint64_t)(c + i) * a.bias_cs];
        }
      }
    }
    if (HIST) count_history<NT == 1024 ? 4 : 2>(a, r0, rows, c0, C, t.classes, 1u, rows * t.classes, lds_words);
#pragma unroll
    for (int u = 0; u < ITER; ++u) {
      if (q[u] >= rows || cl[u] >= C) continue;
      float x[N];
      raw[u].get(x);
      if (HIST) {
        uint32_t w[N], any = 0u;
        __builtin_memcpy(w, __builtin_assume_aligned(lds_words + q[u] * t.classes + cl[u], 16), sizeof(w));
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) any |= w[i];
        if (any) {
#pragma unroll
          for (uint32_t i = 0; i < N; ++i) x[i] = penalise(x[i], w[i], pen[u]);
        }
      }
      if (a.bias) {
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) x[i] += bias[u][i];
      }
#pragma unroll
      for (uint32_t i = 0; i < N; ++i) {
        const uint32_t on = (uint32_t)((int32_t)(bits[u] << (31u - i)) >> 31);
        x[i] = __uint_as_float((__float_as_uint(x[i]) & on) | (0xFF800000u & ~on));
      }
      store_pack<T>(static_cast<T*>(a.out) + (r0 + q[u]) * a.out_stride, c0 + cl[u], a.K, x);
    }
  }
}

// class-major: packs run along the rows of one class; a tile's packs per class are a power of two.  4 M x 10 fp32: 55 us, 5.8 TB/s.
template <class T, bool HIST>
__global__ __launch_bounds__(256) void adjust_classes_kernel(const AdjustArgs a, const AdjustTiles t) {
  constexpr uint32_t N = Pack<T>::N;
  const uint32_t rp = t.rows / N, rp_log2 = 31u - __clz(rp);
  for (uint64_t tile = blockIdx.x; tile < t.tiles; tile += gridDim.x) {
    const uint64_t rt = tile / t.class_tiles, r0 = rt * t.rows;
    const uint32_t c0 = (uint32_t)(tile - rt * t.class_tiles) * t.classes;
    const uint32_t rows = (uint32_t)(a.n - r0 < t.rows ? a.n - r0 : t.rows);
    const uint32_t C = a.K - c0 < t.classes ? a.K - c0 : t.classes;
    if (HIST) count_history<2>(a, r0, rows, c0, C, 1u, t.rows, C * t.rows, lds_words);
    for (uint32_t idx = threadIdx.x; idx < (C << rp_log2); idx += 256u) {
      const uint32_t cl = idx >> rp_log2, rl = (idx & (rp - 1u)) * N, c = c0 + cl;
      if (rl >= rows) continue;
      float x[N];
      load_pack(static_cast<const T*>(a.in) + c * a.in_stride + r0, rl, rows, 0.f, x);
      if (HIST) {
        uint32_t w[N], any = 0u;
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) any |= w[i] = lds_words[cl * t.rows + rl + i];
        if (any) {
#pragma unroll
          for (uint32_t i = 0; i < N; ++i)
            if (w[i]) x[i] = penalise(x[i], w[i], row_penalty(a, r0 + rl + i));
        }
      }
      if (a.bias) {
        const float* b = a.bias + (uint64_t)c * a.bias_cs;
        if (a.bias_rs == 0u) {
          const float v = b[0];
#pragma unroll
          for (uint32_t i = 0; i < N; ++i) x[i] += v;
        } else {
#pragma unroll
          for (uint32_t i = 0; i < N; ++i)
            if (rl + i < rows) x[i] += b[(r0 + rl + i) * a.bias_rs];
        }
      }
      if (a.allowed) {
        const uint32_t* m = a.allowed + (c >> 5);
        if (a.allowed_rs == 0u) {
          const bool on = (m[0] >> (c & 31u)) & 1u;
#pragma unroll
          for (uint32_t i = 0; i < N; ++i) x[i] = on ? x[i] : -kInf;
        } else {
#pragma unroll
          for (uint32_t i = 0; i < N; ++i)
            if (rl + i < rows) x[i] = (m[(r0 + rl + i) * a.allowed_rs] >> (c & 31u)) & 1u ? x[i] : -kInf;
        }
      }
      store_pack(static_cast<T*>(a.out) + c * a.out_stride + r0, rl, rows, x);
    }
  }
}

// ---------------------------------------------------------------------------------------------------
// sums of exponentials: (m, s) = (largest score so far, sum of exp((x - m) / T)).  The difference is taken before the scaling: it is
// finite for finite scores (a row filled with the type's lowest value among them), and small, so exact enough, where it counts.
// A thread's sum runs in 64 bits where its length grows with the row's: fp32 sums of near numbers are all rounded to the same side (one
// score ahead of 2000 alike, added one by one: 500 half steps; 4000: 1000), and they are only as short as the groups that are added here.
// ---------------------------------------------------------------------------------------------------
// of up to 32 exponentials: four chains
template <uint32_t N, class F>
__device__ __forceinline__ float sum_of(F f) {
  float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (uint32_t i = 0; i < N; ++i) t[i & 3u] += f(i);
  return (t[0] + t[1]) + (t[2] + t[3]);
}
struct ExpSum {
  float m = -FLT_MAX, s = 0.f;
  __device__ __forceinline__ void reduce_wave(float c) {  // the same in every lane afterwards
    const float M = wave_max(m);
    s = wave_sum(s * exp2_fast((m - M) * c));
    m = M;
  }
};
// a whole row in one thread, N scores at a time
struct ThreadSum {
  float m = -FLT_MAX;
  double s = 0.0;
  template <uint32_t N>
  __device__ __forceinline__ void add(const float (&x)[N], float c) {
    float pm = x[0];
#pragma unroll
    for (uint32_t i = 1; i < N; ++i) pm = fmaxf(pm, x[i]);
    if (pm > m) {
      s *= (double)exp2_fast((m - pm) * c);
      m = pm;
    }
    s += (double)sum_of<N>([&](uint32_t i) { return exp2_fast((x[i] - m) * c); });
  }
};
// The same, one instruction per score less, for the long rows: exponentials of fma(x, c, -r) with r an fp32 number a step or two above
// m c -- never below it, where 2^(m c - r) of a large score's rounding would overflow.  finish() puts the difference right.  Where that
// rounding is no longer small against 1 (a largest score beyond 10^6 T, or a row without any, whose m is the lowest number) it asks for
// the sum in the plain form instead.
constexpr float kPlainBeyond = 0x1p20f;
template <class S>  // double; float for at most four groups
struct RunSum {
  float m = -FLT_MAX, r;
  S s = 0;
  __device__ __forceinline__ explicit RunSum(float c) : r(reference(-FLT_MAX, c)) {}
  static __device__ __forceinline__ float reference(float m, float c) {
    return fminf(fmaxf(fmaf(fabsf(m * c), 0x1p-23f, m * c), -FLT_MAX), FLT_MAX);
  }
  template <uint32_t M>
  __device__ __forceinline__ float add(const float (&x)[M], float c) {  // -> the largest of x
    float pm = x[0];
#pragma unroll
    for (uint32_t i = 1; i < M; ++i) pm = fmaxf(pm, x[i]);
    if (pm > m) {
      const float nr = reference(pm, c);
      s *= (S)exp2_fast(r - nr);
      m = pm, r = nr;
    }
    s += (S)sum_of<M>([&](uint32_t i) { return exp2_fast(fmaf(x[i], c, -r)); });
    return pm;
  }
  // over the wave, or 16 lanes of it; plain(M) = this lane's sum of exp2((x - M) c)
  template <int LANES, class Plain>
  __device__ __forceinline__ ExpSum finish(float c, Plain plain) const {
    ExpSum e;
    e.m = lanes_max<LANES>(m);
    if (fabsf(e.m * c) <= kPlainBeyond) {
      const float R = reference(e.m, c);
      e.s = lanes_sum<LANES>((float)s * exp2_fast(r - R)) * exp2_fast((float)fma((double)e.m, -(double)c, (double)R));
    } else {
      e.s = lanes_sum<LANES>(plain(e.m));
    }
    return e;
  }
};
template <class Sum>
__device__ __forceinline__ float log_sum(const Sum& e, double inv_T) {
  if (e.m == kInf) return kInf;
  return (float)((double)e.m * inv_T + log_64((double)e.s));  // nothing but -inf: log 0 = -inf
}

// ---------------------------------------------------------------------------------------------------
// top: whole numbers in the order of the scores; 0 = no candidate (NaN, -inf).  -0 and +0 are one score.
// ---------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t score_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return x > -kInf ? b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u) : 0u;
}
__device__ __forceinline__ float key_score(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
// low key bits that are alike for every score of a sign (two-byte types): they need no search
template <class T>
constexpr uint32_t low_bits() {
  return sizeof(T) == 4 ? 0u : __is_same(T, _Float16) ? 13u : 16u;
}
// (key, class) in one number: the larger is the better candidate, equal scores go to the lower class
__device__ __forceinline__ uint64_t candidate(uint32_t key, uint32_t c) { return (uint64_t)key << 32 | (0xFFFFFFFFu - c); }

__device__ __forceinline__ void write_candidate(const TopArgs& a, uint64_t row, uint32_t rank, uint64_t v) {
  a.ids[row * a.k + rank] = (int32_t)(0xFFFFFFFFu - (uint32_t)v);
  a.values[row * a.k + rank] = key_score((uint32_t)(v >> 32));
}
__device__ __forceinline__ void write_nothing(const TopArgs& a, uint64_t row, uint32_t rank) {
  a.ids[row * a.k + rank] = -1;
  a.values[row * a.k + rank] = -kInf;
}

// few classes, few of them wanted: a thread per row, the best k = KK in registers (4 M x 10 fp32 class-major, k = 3: 49 us for 272 MB, 5.5
// TB/s and 42 us' worth of vector issue).  Row-major rows are staged in LDS (coalesced loads; the row pitch is an odd number of words),
// class-major ones are coalesced as they are.
template <class T>
__device__ __forceinline__ uint32_t staged_pitch(uint32_t K) {  // elements
  constexpr uint32_t per_word = 4 / sizeof(T);
  return (((K + per_word - 1) / per_word) | 1u) * per_word;
}
template <class T>
__device__ __forceinline__ void stage_rows(const T* in, uint64_t r0, uint32_t rows, uint32_t K, uint64_t stride, T* dst, uint32_t pitch) {
  if (stride == K) {  // one piece of rows * K scores (at most 256 * 64)
    const T* src = in + r0 * K;
    const uint32_t total = rows * K, magic = (uint32_t)((0x100000000ull + K - 1u) / K);  // K >= 2: i / K = umulhi(i, magic) for i < 2^16
    constexpr uint32_t N = Pack<T>::N;
    for (uint32_t i = threadIdx.x * N; i < total; i += 256u * N) {
      uint32_t r = K == 1u ? i : __umulhi(i, magic), c = i - r * K;
      typename Pack<T>::vec v;
      if (i + N <= total) __builtin_memcpy(&v, src + i, 16);
      else {
#pragma unroll
        for (uint32_t j = 0; j < N; ++j) v[j] = i + j < total ? src[i + j] : (T)0.f;
      }
#pragma unroll
      for (uint32_t j = 0; j < N; ++j) {
        if (i + j < total) dst[r * pitch + c] = v[j];
        if (++c == K) c = 0u, ++r;
      }
    }
  } else {
    for (uint32_t r = threadIdx.x >> 5; r < rows; r += 8u)
      for (uint32_t c = threadIdx.x & 31u; c < K; c += 32u) dst[r * pitch + c] = in[(r0 + r) * stride + c];
  }
}

template <class T, bool CM, int KK>
__global__ __launch_bounds__(256) void top_thread_kernel(const TopArgs a) {
  T* stage = reinterpret_cast<T*>(lds_words);
  const uint32_t pitch = staged_pitch<T>(a.K);
  const float c2 = a.scale;
  const uint64_t step = (uint64_t)gridDim.x * 256u;
  for (uint64_t r0 = (uint64_t)blockIdx.x * 256u; r0 < a.n; r0 += step) {
    const uint32_t rows = (uint32_t)(a.n - r0 < 256u ? a.n - r0 : 256u);
    const T* in = static_cast<const T*>(a.in);
    if (!CM) {
      __syncthreads();
      stage_rows(in, r0, rows, a.K, a.stride, stage, pitch);
      __syncthreads();
    }
    const uint32_t tid = forgotten(threadIdx.x);
    if (tid >= rows) continue;
    const uint64_t row = r0 + tid;
    float v[KK];
    int32_t id[KK];
#pragma unroll
    for (int j = 0; j < KK; ++j) v[j] = -kInf, id[j] = -1;
    ThreadSum e;
    constexpr uint32_t kAhead = 8;  // scores of a row that are summed together; class-major: their loads in flight
    for (uint32_t c0 = 0; c0 < a.K; c0 += kAhead) {
      T next[kAhead];
#pragma unroll
      for (uint32_t i = 0; i < kAhead; ++i) next[i] = c0 + i >= a.K ? (T)-kInf : CM ? in[(c0 + i) * a.stride + row] : stage[tid * pitch + c0 + i];
      float xs[kAhead];
#pragma unroll
      for (uint32_t i = 0; i < kAhead; ++i) xs[i] = (float)next[i];
      e.add(xs, c2);
#pragma unroll
      for (uint32_t i = 0; i < kAhead; ++i) {
        float x = xs[i];
        if (x > v[KK - 1]) {  // (false for NaN and -inf)
          int32_t xi = (int32_t)(c0 + i);
          bool placed = false;
#pragma unroll
          for (int j = 0; j < KK; ++j) {  // equal scores: the class that came first stays in front
            placed |= x > v[j];
            const float tv = v[j];
            const int32_t ti = id[j];
            v[j] = placed ? x : tv, id[j] = placed ? xi : ti;
            x = placed ? tv : x, xi = placed ? ti : xi;
          }
        }
      }
    }
    __builtin_memcpy(a.ids + row * KK, id, sizeof(id));  // (one store: a wave writes one piece)
    __builtin_memcpy(a.values + row * KK, v, sizeof(v));
    if (a.lse) a.lse[row] = log_sum(e, a.inv_T);
  }
}

// A number that at least kk of the keys in a wave's registers (E per lane) reach: greedy from the top bit, counted with ballots.  Bits
// below the 16th (sign, exponent and 7 bits of a score) are looked at only while more than kk + slack keys reach it: slack 0 and keys that
// tie across kk give the kk-th largest key itself.  Fewer keys than kk: 0.
template <int E>
__device__ __forceinline__ uint32_t wave_kth_key(const uint32_t (&key)[E], uint32_t kk, uint32_t slack, uint32_t low) {
  uint32_t t = 0u, reach = 64u * E;
  for (int bit = 31; bit >= (int)low; --bit) {
    if (bit < 16 && reach <= kk + slack) break;
    const uint32_t cand = t | (1u << bit);
    uint32_t cnt = 0u;
#pragma unroll
    for (int i = 0; i < E; ++i) cnt += __popcll(__ballot(key[i] >= cand));
    if (cnt >= kk) {
      t = cand, reach = cnt;
      if (cnt == kk) break;
    }
  }
  return t;
}
// how many of `count` candidates in LDS are better than `mine`
__device__ __forceinline__ uint32_t rank_of(uint64_t mine, const uint64_t* list, uint32_t count) {
  uint32_t rank = 0u;
#pragma unroll 8
  for (uint32_t j = 0; j < count; ++j) rank += list[j] > mine;
  return rank;
}

// few classes, more than 8 of them wanted: a thread per row, every class's rank counted against the others'.  For c < d one comparison
// serves both: g = x_d > x_c puts d before c, otherwise c, the lower class, stands first.  KP >= K classes in registers.
template <class T, bool CM, int KP>
__global__ __launch_bounds__(256) void top_rank_kernel(const TopArgs a) {
  T* stage = reinterpret_cast<T*>(lds_words);
  const uint32_t pitch = staged_pitch<T>(a.K), columns = a.k < a.K ? a.k : a.K, opitch = columns | 1u;
  float* out_value = reinterpret_cast<float*>(lds_words);  // (takes the place of the staged rows, which are in registers by then)
  int32_t* out_id = reinterpret_cast<int32_t*>(lds_words + 256u * opitch);
  const float c2 = a.scale;
  for (uint64_t r0 = (uint64_t)blockIdx.x * 256u; r0 < a.n; r0 += (uint64_t)gridDim.x * 256u) {
    const uint32_t rows = (uint32_t)(a.n - r0 < 256u ? a.n - r0 : 256u), tid = forgotten(threadIdx.x);
    const T* in = static_cast<const T*>(a.in);
    const bool active = tid < rows;
    __syncthreads();
    if (!CM) {
      stage_rows(in, r0, rows, a.K, a.stride, stage, pitch);
      __syncthreads();
    }
    float x[KP];
    if (active) {
#pragma unroll
      for (uint32_t c = 0; c < KP; ++c) x[c] = c < a.K ? (float)(CM ? in[c * a.stride + r0 + tid] : stage[tid * pitch + c]) : -kInf;
    }
    __syncthreads();
    if (active) {
      ExpSum e;
#pragma unroll
      for (int c = 0; c < KP; ++c) e.m = fmaxf(e.m, x[c]);
#pragma unroll
      for (int c = 0; c < KP; ++c) {
        e.s += exp2_fast((x[c] - e.m) * c2);
        x[c] = x[c] > -kInf ? x[c] : -kInf;  // (NaN is no candidate)
      }
      if (a.lse) a.lse[r0 + tid] = log_sum(e, a.inv_T);
      uint32_t rank[KP];
#pragma unroll
      for (int c = 0; c < KP; ++c) rank[c] = c;
#pragma unroll
      for (int c = 0; c < KP; ++c)
#pragma unroll
        for (int d = c + 1; d < KP; ++d) {
          const bool g = x[d] > x[c];
          rank[c] += g, rank[d] -= g;
        }
      float* ov = out_value + tid * opitch;
      int32_t* oi = out_id + tid * opitch;
      for (uint32_t j = 0; j < columns; ++j) ov[j] = -kInf, oi[j] = -1;
#pragma unroll
      for (int c = 0; c < KP; ++c)
        if (x[c] > -kInf && rank[c] < columns) ov[rank[c]] = x[c], oi[rank[c]] = c;
    }
    __syncthreads();
    const uint32_t total = rows * a.k, magic = 0xFFFFFFFFu / a.k + 1u;  // (total k < 2^32, k > 8)
    for (uint32_t i = tid; i < total; i += 256u) {
      const uint32_t r = __umulhi(i, magic), j = i - r * a.k;
      a.ids[r0 * a.k + i] = j < columns ? out_id[r * opitch + j] : -1;
      a.values[r0 * a.k + i] = j < columns ? out_value[r * opitch + j] : -kInf;
    }
  }
}

// class-major rows [r0, r0 + 16) into stage[class][17] as fp32: 64-byte pieces (of fp32) out of every class's vector; with 17 words per class
// neither the writes nor reads by consecutive lanes of consecutive classes meet in a bank
constexpr uint32_t kStagePitch = 17;
template <class T>
__device__ __forceinline__ void stage_class_major(const TopArgs& a, uint64_t r0, float* stage) {
  constexpr uint32_t N = Pack<T>::N, kPieces = 16u / N;
  const uint32_t rows = (uint32_t)(a.n - r0 < 16u ? a.n - r0 : 16u), q = threadIdx.x % kPieces * N;
  for (uint32_t c = threadIdx.x / kPieces; c < a.K; c += blockDim.x / kPieces) {
    float v[N];
    load_pack(static_cast<const T*>(a.in) + c * a.stride + r0, q, rows, 0.f, v);
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) stage[c * kStagePitch + q + i] = v[i];
  }
}

// short rows, few classes wanted: 16 lanes per row, P packs per lane in registers; the best is taken out k times, lane j keeps the j-th.
template <class T, bool CM, int P>
__global__ __launch_bounds__(256) void top_lanes_kernel(const TopArgs a) {
  constexpr int N = (int)Pack<T>::N, E = P * N;
  float* stage = reinterpret_cast<float*>(lds_words);
  const float c2 = a.scale;
  for (uint64_t r0 = (uint64_t)blockIdx.x * 16u; r0 < a.n; r0 += (uint64_t)gridDim.x * 16u) {
    if (CM) {
      __syncthreads();
      stage_class_major<T>(a, r0, stage);
      __syncthreads();
    }
    const uint64_t row = r0 + (threadIdx.x >> 4);
    if (row >= a.n) continue;
    const uint32_t lane = forgotten(threadIdx.x & 15u);
    float x[E], best = -kInf;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      float v[N];
      if (CM) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const uint32_t c = (uint32_t)(p * N + i) * 16u + lane;
          v[i] = c < a.K ? stage[c * kStagePitch + (threadIdx.x >> 4)] : -kInf;
        }
      } else {
        load_pack(static_cast<const T*>(a.in) + row * a.stride, ((uint32_t)p * 16u + lane) * N, a.K, -kInf, v);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) x[p * N + i] = v[i], best = fmaxf(best, v[i]);
    }
    ExpSum e;
    e.m = fmaxf(lanes_max<16>(best), -FLT_MAX);
#pragma unroll
    for (int i = 0; i < E; ++i) e.s += exp2_fast((x[i] - e.m) * c2);
    e.s = lanes_sum<16>(e.s);
    if (a.lse && lane == 0u) a.lse[row] = log_sum(e, a.inv_T);
    float value = -kInf;
    int32_t id = -1;
    for (uint32_t j = 0; j < a.k; ++j) {
      float b = -kInf;
      uint32_t at = 0xFFFFFFFFu;
#pragma unroll
      for (int i = 0; i < E; ++i) {  // (in the order of the classes; NaN and -inf are never better)
        const bool g = x[i] > b;
        b = g ? x[i] : b, at = g ? (uint32_t)i : at;
      }
      const uint32_t mine = at == 0xFFFFFFFFu ? at : CM ? at * 16u + lane : (at / N * 16u + lane) * N + at % N;
      uint32_t c = mine;
      auto meet = [&](float ob, uint32_t oc) {
        const bool g = ob > b || (ob == b && oc < c);
        b = g ? ob : b, c = g ? oc : c;
      };
      meet(dpp<kRowRor8, 0xF>(b, b), dpp<kRowRor8, 0xF>(c, c));
      meet(dpp<kRowRor4, 0xF>(b, b), dpp<kRowRor4, 0xF>(c, c));
      meet(dpp<kRowRor2, 0xF>(b, b), dpp<kRowRor2, 0xF>(c, c));
      meet(dpp<kRowRor1, 0xF>(b, b), dpp<kRowRor1, 0xF>(c, c));
      if (lane == j) value = b, id = (int32_t)c;  // (nothing left: -inf and -1)
      if (c == mine) {
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = (uint32_t)i == at ? -kInf : x[i];
      }
    }
    if (lane < a.k) a.ids[row * a.k + lane] = id, a.values[row * a.k + lane] = value;
  }
}

// up to 2048 classes: a wave per row, all its scores in registers (P packs per lane).  16384 x 1000 fp32, k = 20: 24 us.  What bounds it is
// neither the 65 MB nor the 519 vector instructions per row (14 us' worth of issue) but a wave's chain of dependent steps: the bits of the
// bound, the list, the ranks.  Class-major rows are staged through LDS, 16 at a time for the 8 waves of the block.
constexpr uint32_t kWaveList = 128;  // candidates that are ranked without an exact count
__device__ __forceinline__ uint32_t lanes_below(uint64_t ballot) {
  return __builtin_amdgcn_mbcnt_hi((uint32_t)(ballot >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)ballot, 0u));
}
__host__ __device__ constexpr uint32_t wave_list(uint32_t k) { return k > kWaveList ? k : kWaveList; }
constexpr uint32_t top_wave_rows(bool class_major) { return class_major ? 16u : 4u; }
constexpr uint32_t top_wave_waves(bool class_major) { return class_major ? 8u : 4u; }
template <class T, bool CM, int P>
__global__ __launch_bounds__(top_wave_waves(CM) * 64) void top_wave_kernel(const TopArgs a) {
  constexpr int N = (int)Pack<T>::N, E = P * N;
  constexpr uint32_t kRows = top_wave_rows(CM), kWaves = top_wave_waves(CM);
  const uint32_t wave = threadIdx.x >> 6;
  uint64_t* list = reinterpret_cast<uint64_t*>(lds_words) + wave * wave_list(a.k);  // the wave's selected candidates
  float* stage = reinterpret_cast<float*>(reinterpret_cast<uint64_t*>(lds_words) + kWaves * wave_list(a.k));  // class-major
  const float c2 = a.scale;
  for (uint64_t r0 = (uint64_t)blockIdx.x * kRows; r0 < a.n; r0 += (uint64_t)gridDim.x * kRows) {
    if (CM) {
      __syncthreads();
      stage_class_major<T>(a, r0, stage);
      __syncthreads();
    }
    for (uint32_t rr = wave; rr < kRows && r0 + rr < a.n; rr += kWaves) {
      const uint64_t row = r0 + rr;
      const uint32_t lane = forgotten(threadIdx.x & 63u);
      auto class_of = [&](int i) { return CM ? (uint32_t)i * 64u + lane : ((uint32_t)(i / N) * 64u + lane) * N + i % N; };
      float x[E];
      float best = -kInf;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        float v[N];
        if (CM) {
#pragma unroll
          for (int i = 0; i < N; ++i) v[i] = class_of(p * N + i) < a.K ? stage[class_of(p * N + i) * kStagePitch + rr] : -kInf;
        } else {
          load_pack(static_cast<const T*>(a.in) + row * a.stride, class_of(p * N), a.K, -kInf, v);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) x[p * N + i] = v[i], best = fmaxf(best, v[i]);
      }
      ExpSum e;
      e.m = fmaxf(wave_max(best), -FLT_MAX);
#pragma unroll
      for (int i = 0; i < E; ++i) e.s += exp2_fast((x[i] - e.m) * c2);
      e.s = wave_sum(e.s);
      if (a.lse && lane == 0u) a.lse[row] = log_sum(e, a.inv_T);
      // A bound that at least k scores reach: the k-th largest of the lanes' best, or a little below it.  What reaches it is listed and
      // ranked.
      uint32_t count = kWaveList + 1u;
      if (a.k <= 64u) {
        const uint32_t lane_key[1] = {score_key(best)};
        const uint32_t t = wave_kth_key(lane_key, a.k, a.k, low_bits<T>());
        const float bound = t ? key_score(t) : -FLT_MAX;
        count = 0u;
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const bool take = x[i] >= bound;
          const uint64_t b = __ballot(take);
          const uint32_t slot = count + lanes_below(b);
          if (take && slot < kWaveList) list[slot] = (uint64_t)__float_as_uint(x[i]) << 32 | class_of(i);
          count += __popcll(b);
        }
        if (count <= kWaveList) {  // scores and classes to candidates: once per candidate, not once per place that might hold one
          __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
          __builtin_amdgcn_wave_barrier();
          for (uint32_t i = lane; i < count; i += 64u) {
            const uint64_t v = list[i];
            list[i] = candidate(score_key(__uint_as_float((uint32_t)(v >> 32))), (uint32_t)v);
          }
        }
      }
      if (count > kWaveList) {  // many wanted, or many that tie: count exactly, bit by bit
        uint32_t key[E];
        uint32_t valid = 0u;
#pragma unroll
        for (int i = 0; i < E; ++i) key[i] = score_key(x[i]), valid += __popcll(__ballot(key[i] != 0u));
        const uint32_t kk = valid < a.k ? valid : a.k;
        uint32_t t = wave_kth_key(key, kk, 0u, low_bits<T>());
        if (t == 0u) t = 1u;  // (fewer than k candidates: all of them)
        // everything from t up, if that is kk; else what lies above t's score, and of the classes with t's score the lowest ones
        uint32_t ge = 0u, gt = 0u;
        const uint32_t above = t + (1u << low_bits<T>());
#pragma unroll
        for (int i = 0; i < E; ++i) ge += __popcll(__ballot(key[i] >= t)), gt += __popcll(__ballot(key[i] >= above));
        uint32_t last = 0xFFFFFFFFu;  // highest class admitted among the equal ones
        if (ge > kk) {
          last = 0u;
          for (int bit = 10; bit >= 0; --bit) {  // (at most 2048 classes)
            const uint32_t cand = last + (1u << bit);
            uint32_t cnt = gt;
#pragma unroll
            for (int i = 0; i < E; ++i) {
              const uint32_t c = class_of(i);
              cnt += __popcll(__ballot(key[i] >= t && key[i] < above && c < cand));
            }
            if (cnt < kk) last = cand;
          }
        }
        count = 0u;
#pragma unroll
        for (int i = 0; i < E; ++i) {
          const uint32_t c = class_of(i);
          const bool take = key[i] >= t && (key[i] >= above || c <= last);
          const uint64_t b = __ballot(take);
          if (take) list[count + lanes_below(b)] = candidate(key[i], c);
          count += __popcll(b);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      for (uint32_t i = lane; i < (count > a.k ? count : a.k); i += 64u) {
        if (i >= count) {
          write_nothing(a, row, i);
          continue;
        }
        const uint64_t mine = list[i];
        const uint32_t rank = rank_of(mine, list, count);
        if (rank < a.k) write_candidate(a, row, rank, mine);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();  // the next row's candidates go into the same list
    }
  }
}

// many classes: a block of NT threads per row, four packs of a thread at a time (a chunk).  One pass keeps the sum of exponentials, the
// thread's largest score, and the largest score of each group of chunks (at most 16 groups; to 16 bits, in LDS).  The k-th largest of the
// threads' maxima is a bound that at least k scores reach, and only the groups that reach it -- about k of them, 64 packs of
// 128000 -- are read a second time to list the candidates.  Rows with more candidates than the list holds (scores that tie, or stand
// in few threads) are narrowed down by counting, bit by bit, over the threads that reach the bound.
// 512 x 128000 bf16, k = 64: 30 us for 131 MB, 22 of them reading at the 6 TB/s of a plain read; bound, second look and ranks of the two rows
// of a CU come behind it with nothing to hide them.  With a second look at every pack of the threads that hold candidates -- a cache line each, the
// whole row over -- it was 41.
constexpr uint32_t kListCap = 1024, kGroups = 16;
constexpr uint32_t top_block_words(uint32_t threads) {  // LDS
  return 2u * kListCap + threads + 2u * (threads / 64u) + 4u + threads / 64u + kGroups * threads / 2u;
}
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, true));
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, true));
}
template <class T, int NT>
__global__ __launch_bounds__(NT) void top_block_kernel(const TopArgs a) {
  constexpr uint32_t N = Pack<T>::N, kWaves = NT / 64;
  uint64_t* list = reinterpret_cast<uint64_t*>(lds_words);         // [kListCap]
  uint32_t* maxima = lds_words + 2 * kListCap;                     // [NT]
  float* part = reinterpret_cast<float*>(maxima + NT);             // [2 * kWaves]
  uint32_t* ctl = reinterpret_cast<uint32_t*>(part + 2 * kWaves);  // [0] bound, [1] candidates, [2] groups that hold them, [4 ..] counts per wave
  uint16_t* group_max = reinterpret_cast<uint16_t*>(ctl + 4 + kWaves);  // [kGroups][NT]
  const uint32_t packs = (a.K + N - 1u) / N, chunks = (packs + 4u * NT - 1u) / (4u * NT);
  const uint32_t per_group = (chunks + kGroups - 1u) / kGroups;  // chunks
  const float c2 = a.scale;
  for (uint64_t row = blockIdx.x; row < a.n; row += gridDim.x) {
    const T* in = static_cast<const T*>(a.in) + row * a.stride;
    const uint32_t tid = forgotten(threadIdx.x), lane = tid & 63u, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    RunSum<double> run(c2);
    float largest = -kInf;  // of the group
    uint32_t p0 = 0, groups = 0, left = per_group;
    __syncthreads();  // the row before is written
    auto chunk_done = [&](float pm) {
      largest = fmaxf(largest, pm);
      if (--left == 0u) {
        group_max[groups * NT + tid] = (uint16_t)(score_key(largest) >> 16);
        ++groups, left = per_group, largest = -kInf;
      }
    };
    for (; (p0 + 4u * NT) * N <= a.K; p0 += 4u * NT) {
      float x[4 * N];
      load_packs<T, NT>(in, p0 + tid, x);
      chunk_done(run.add(x, c2));
    }
    if (p0 < packs) {
      float pm = -kInf;
      if (p0 + tid < packs) {
        float x[4 * N];
        load_last_packs<T, NT>(in, p0 + tid, a.K, -kInf, x);
        pm = run.add(x, c2);
      }
      left = 1u;
      chunk_done(pm);
    } else if (left != per_group) {
      left = 1u;
      chunk_done(-kInf);
    }
    const uint32_t best = score_key(run.m);  // (a thread without a candidate counts with the lowest score: the bound only sinks)
    const ExpSum e = run.finish<64>(c2, [&](float M) {
      double t = 0.0;
      for (uint32_t p = tid; p < packs; p += NT) {
        float x[N];
        load_pack(in, p * N, a.K, -kInf, x);
        t += (double)sum_of<N>([&](uint32_t i) { return exp2_fast((x[i] - M) * c2); });
      }
      return (float)t;
    });
    const bool quads = a.k <= NT / 8u;  // few wanted: the largest of four lanes will do, and is a quarter to search
    if (quads) {
      const uint32_t q = quad_max(best);
      if ((tid & 3u) == 0u) maxima[tid >> 2] = q;
    } else {
      maxima[tid] = best;
    }
    if (lane == 0u) part[2 * wave] = e.m, part[2 * wave + 1] = e.s;
    if (tid == 0u) ctl[1] = 0u, ctl[2] = 0u;
    __syncthreads();
    if (wave == 0u) {
      uint32_t t;
      if (quads) {
        uint32_t key[NT / 256];
#pragma unroll
        for (int i = 0; i < NT / 256; ++i) key[i] = maxima[i * 64 + lane];
        t = wave_kth_key(key, a.k, a.k / 4u, low_bits<T>());
      } else {
        uint32_t key[NT / 64];
#pragma unroll
        for (int i = 0; i < NT / 64; ++i) key[i] = maxima[i * 64 + lane];
        t = wave_kth_key(key, a.k, a.k / 4u, low_bits<T>());
      }
      if (lane == 0u) ctl[0] = t ? t : 1u;
    } else if (wave == 1u && a.lse) {
      ExpSum w;
      w.m = lane < kWaves ? part[2 * lane] : -FLT_MAX, w.s = lane < kWaves ? part[2 * lane + 1] : 0.f;
      w.reduce_wave(c2);
      if (lane == 0u) a.lse[row] = log_sum(w, a.inv_T);
    }
    __syncthreads();
    const uint32_t bound = ctl[0];
    const bool mine = best >= bound;
    uint32_t* owners = maxima;  // group * NT + thread, of the groups that hold candidates
    if (mine)
      for (uint32_t g = 0; g < groups; ++g)
        if (group_max[g * NT + tid] >= bound >> 16) {
          const uint32_t slot = atomicAdd(&ctl[2], 1u);
          if (slot < NT) owners[slot] = g * NT + tid;
        }
    __syncthreads();
    auto look = [&](const float (&x)[N], uint32_t c) {
#pragma unroll
      for (uint32_t j = 0; j < N; ++j) {
        const uint32_t key = score_key(x[j]);
        if (key >= bound) {
          const uint32_t slot = atomicAdd(&ctl[1], 1u);
          if (slot < kListCap) list[slot] = candidate(key, c + j);
        }
      }
    };
    if (ctl[2] <= NT) {
      // their packs, dealt out over the whole block: item i = pack (i mod per) of owner (i div per)
      const uint32_t per = 4u * per_group, items = ctl[2] * per, magic = 0xFFFFFFFFu / per + 1u;  // (i per < 2^32, per >= 4)
      for (uint32_t i = tid; i < items; i += NT) {
        const uint32_t o = __umulhi(i, magic), own = owners[o], g = own / NT;
        const uint32_t c = ((g * per + i - o * per) * NT + own % NT) * N;
        float x[N];
        load_pack(in, c, a.K, -kInf, x);
        look(x, c);
      }
    } else if (mine) {
      for (uint32_t p = tid; p < packs; p += NT) {
        float x[N];
        load_pack(in, p * N, a.K, -kInf, x);
        look(x, p * N);
      }
    }
    __syncthreads();
    uint32_t count = ctl[1];
    if (count > kListCap) {
      const uint32_t kk = count < a.k ? count : a.k;
      // candidates in [lo, hi) with class < below, over the whole block
      auto count_if = [&](uint32_t lo, uint32_t hi, uint32_t below) -> uint32_t {
        uint32_t n = 0u;
        if (mine)
          for (uint32_t p = tid; p < packs; p += NT) {
            float x[N];
            load_pack(in, p * N, a.K, -kInf, x);
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) {
              const uint32_t key = score_key(x[i]);
              n += key >= lo && key < hi && p * N + i < below;
            }
          }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) n += __shfl_xor(n, d);
        __syncthreads();
        if (lane == 0u) ctl[4 + wave] = n;
        __syncthreads();
        uint32_t sum = 0u;
        for (uint32_t w = 0; w < kWaves; ++w) sum += ctl[4 + w];
        return sum;
      };
      uint32_t t = bound;  // raised to the kk-th largest key: bits below the bound's differing ones are tried from the top
      {
        uint32_t v = 0u;
        for (int bit = 31; bit >= (int)low_bits<T>(); --bit) {
          const uint32_t cand = v | (1u << bit);
          if (cand <= bound || count_if(cand, 0xFFFFFFFFu, 0xFFFFFFFFu) >= kk) v = cand;
        }
        if (v > t) t = v;
      }
      const uint32_t above = t + (1u << low_bits<T>());
      const uint32_t gt = count_if(above, 0xFFFFFFFFu, 0xFFFFFFFFu);
      uint32_t last = 0u;
      for (int bit = 19; bit >= 0; --bit) {  // (at most 2^20 classes)
        const uint32_t cand = last + (1u << bit);
        if (gt + count_if(t, above, cand) < kk) last = cand;
      }
      __syncthreads();
      if (tid == 0u) ctl[1] = 0u;
      __syncthreads();
      if (mine)
        for (uint32_t p = tid; p < packs; p += NT) {
          float x[N];
          load_pack(in, p * N, a.K, -kInf, x);
#pragma unroll
          for (uint32_t i = 0; i < N; ++i) {
            const uint32_t key = score_key(x[i]), c = p * N + i;
            if (key >= above || (key >= t && c <= last)) list[atomicAdd(&ctl[1], 1u) & (kListCap - 1u)] = candidate(key, c);
          }
        }
      __syncthreads();
      count = ctl[1];
    }
    for (uint32_t i = tid; i < (count > a.k ? count : a.k); i += NT) {
      if (i >= count) {
        write_nothing(a, row, i);
        continue;
      }
      const uint64_t v = list[i];
      const uint32_t rank = rank_of(v, list, count);
      if (rank < a.k) write_candidate(a, row, rank, v);
    }
  }
}

// ---------------------------------------------------------------------------------------------------
// distill.  With z = student / T, S = the listed classes, m_o, s_o = (largest score, sum of exp((x - m_o) / T)) over the classes OUTSIDE
// S, and everything of a row's own (2 k exponentials) in 64 bits:
//   Z = s_o e^((m_o - M) / T) + sum_S e^((x_c - M) / T),  p_R = its first summand / Z,  log p_c = (x_c - M) / T - log Z
//   loss = sum_j q_j (log q_j - log p_(i_j)) + q_R (log q_R - log p_R)
//   gradient outside S: p_c (Q - q_R / p_R) = e^((x_c - m_o) / T) * [(Q p_R - q_R) / s_o]     (one coefficient per row)
//   gradient inside S:  p_c Q - sum of the class's q_j                                        (at most k per row)
// The sums are kept apart because 1 - sum_S p and a loss near zero are differences of near numbers: p_R comes from its own sum, and an
// error of s_o moves all p together so that it enters the loss times (p_R - q_R) only.
// ---------------------------------------------------------------------------------------------------
// Is the teacher's rest 1 - Q more than the rounding of its log-sum-exp (half a step, and 200 of them in the sum that it came from)?  Asked
// only where the student has no probability for it: the loss is infinite then, and no loss at all if the teacher's rest is 0.
__device__ __forceinline__ bool rest_counts(double Q, float lse) { return (float)(1.0 - Q) > (256.f + fabsf(lse)) * 0x1p-24f; }

// what the gradient's pass over the row needs: grad = coef * exp((x - m) / T) outside S
struct RowGrad {
  float m, coef;
};

constexpr int32_t kAgain = 1 << 30;  // on a class number: an earlier entry of the row lists the class already

// a row's entries in LDS (k of each): e^((x - M) / T) of the student, the teacher's probability, the class (-1 = no entry), both scores
struct Entries {
  double *e, *q;
  int32_t* id;
  float *x, *t;
  __device__ explicit Entries(uint32_t* base, uint32_t k) {
    e = reinterpret_cast<double*>(base), q = e + k, id = reinterpret_cast<int32_t*>(q + k), x = reinterpret_cast<float*>(id + k), t = x + k;
  }
  static __host__ __device__ constexpr uint32_t words(uint32_t k) { return 7u * k; }
};

// one wave (or L = 16 lanes of it), one row: the teacher's entries against the student's row.  o = sums outside S, a bitmap.
template <class T, int L, bool GRAD>
__device__ __forceinline__ RowGrad row_loss(const DistillArgs& a, uint64_t row, const Entries& en, const uint32_t* S, uint32_t lane,
                                            const ExpSum& o) {
  // the student's scale is the fp32 one of the sums outside S, for all its classes: p stays a softmax, of a temperature off by 2^-25
  const double inv_T = a.inv_T, x_scale = (double)a.scale;
  constexpr double kLn2 = 0.69314718055994530942;
  float xm = -FLT_MAX, tm = -FLT_MAX;
  for (uint32_t j = lane; j < a.k; j += L)
    if (en.id[j] >= 0) xm = fmaxf(xm, en.x[j]), tm = fmaxf(tm, en.t[j]);
  const float M = lanes_max<L>(fmaxf(xm, o.m));
  tm = lanes_max<L>(tm);
  const double shift = a.lse ? (double)a.lse[row] : (double)tm * inv_T;
  double zs = 0.0, ts = 0.0;
  for (uint32_t j = lane; j < a.k; j += L)
    if (en.id[j] >= 0) {
      const double e = exp2_64(((double)en.x[j] - (double)M) * x_scale), q = exp2_64(((double)en.t[j] * inv_T - shift) * kLog2e);
      en.e[j] = e, en.q[j] = q;
      ts += q;
      if (!(en.id[j] & kAgain)) zs += e;
    }
  zs = lanes_sum<L>(zs), ts = lanes_sum<L>(ts);
  const double far = exp2_64(((double)o.m - (double)M) * x_scale), Z = (double)o.s * far + zs, log_Z = log_64(Z);
  // without lse the q are still to be divided by their sum
  const double log_T = a.lse ? shift : shift + log_64(ts), scale = a.lse ? 1.0 : inverse_64(ts);
  double Q = a.lse ? ts : ts * scale, rest_s = 0.0, loss = 0.0;  // (1 without lse, or NaN); rest_s = q_R / s_o
  for (uint32_t j = lane; j < a.k; j += L)
    if (en.id[j] >= 0 && !(en.q[j] == 0.0))
      loss += en.q[j] * scale * (((double)en.t[j] * inv_T - log_T) - (((double)en.x[j] - (double)M) * x_scale * kLn2 - log_Z));
  loss = lanes_sum<L>(loss);
  if (a.lse && o.s > 0.f && Q < 1.0) {
    rest_s = (1.0 - Q) * inverse_64((double)o.s);
    loss += (1.0 - Q) * (log_64(rest_s) - (((double)o.m - (double)M) * x_scale * kLn2 - log_Z));
    Q = 1.0;
  }
  // a student's row without a softmax (NaN, +inf, or nothing but -inf), or a teacher's: also where no entry's probability carries it on
  const bool none = !(Z > 0.0 && Q >= 0.0 && Q < __builtin_inf());
  if (a.loss && lane == 0u) {
    float v = none ? __builtin_nanf("") : (float)loss;
    if (o.s == 0.f && a.lse && rest_counts(Q, a.lse[row])) {
      uint32_t listed = 0u;
      for (uint32_t i = 0; a.K <= a.k && i < (a.K + 31u) / 32u; ++i) listed += __popc(S[i]);
      if (listed < a.K) v += kInf;
    }
    a.loss[row] = v;
  }
  RowGrad g = {o.m, 0.f};
  if (GRAD) {
    const double w = (a.weight ? (double)a.weight[row * a.weight_stride] : 1.0) * inv_T;
    const double p_scale = none ? __builtin_nan("") : Q * inverse_64(Z);
    g.coef = o.s == 0.f && !none ? 0.f : (float)((p_scale * far - rest_s) * w);  // (nothing outside S: no gradient there)
    T* out = static_cast<T*>(a.grad) + row * a.grad_stride;
    for (uint32_t j = lane; j < a.k; j += L) {
      const int32_t id = en.id[j];
      if (id < 0 || (id & kAgain)) continue;
      double qc = en.q[j];
      for (uint32_t i = j + 1u; i < a.k; ++i)  // further entries of this class, in their order
        if (en.id[i] == (id | kAgain)) qc += en.q[i];
      out[id] = (T)(float)((en.e[j] * p_scale - qc * scale) * w);
    }
  }
  return g;
}

__host__ __device__ constexpr uint32_t distill_words(uint32_t K, uint32_t k, uint32_t threads) {  // LDS of a row, an even number
  return (Entries::words(k) + 4u + 2u * ((threads + 63u) / 64u) + (K + 31u) / 32u + 1u) & ~1u;
}

// NT threads per row: 16 (4 rows per wave: what a row does once costs a fourth of a wave), 64 (a wave) or the whole block.  P > 0: the
// row's packs stay in registers, P per thread, all of them loaded at once while the teacher's entries are fetched, so that the gradient
// costs one read and one write of the matrix.
// P = 0 (rows of more than 512 x 32 packs): the row is read a second time for the gradient, from whichever cache still holds it.
// S is a bitmap in LDS, a pack's bits next to each other.
template <class T, int NT, int P, bool GRAD>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void distill_kernel(const DistillArgs a) {
  constexpr uint32_t N = Pack<T>::N, kGroups = NT < 256 ? 256 / NT : 1, kWaves = (NT + 63) / 64, kFull = (1u << N) - 1u;
  const uint32_t group = NT < 256 ? threadIdx.x / NT : 0u;
  const uint32_t words = (a.K + 31u) / 32u;
  uint32_t* base = lds_words + group * distill_words(a.K, a.k, NT);
  const Entries en(base, a.k);
  uint32_t* ctl = base + Entries::words(a.k);            // [0] any entry, [1] any class twice, [2, 3] RowGrad
  float* part = reinterpret_cast<float*>(ctl + 4);       // [2 * kWaves]
  uint32_t* bitmap = ctl + 4 + 2u * kWaves;              // [words]
  const uint32_t packs = (a.K + N - 1u) / N;
  const float c2 = a.scale;
  auto sync = [] {
    if (NT <= 64) {
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    } else {
      __syncthreads();
    }
  };
  auto listed_bits = [&](uint32_t p) { return bitmap[p * N >> 5] >> (p * N & 31u) & kFull; };
  for (uint64_t row = (uint64_t)blockIdx.x * kGroups + group; row < a.n; row += (uint64_t)gridDim.x * kGroups) {
    const T* in = static_cast<const T*>(a.in) + row * a.stride;
    T* out = static_cast<T*>(a.grad) + row * a.grad_stride;
    const uint32_t tid = forgotten(NT < 256 ? threadIdx.x % NT : threadIdx.x), lane = tid & 63u;
    sync();  // the row before is done with the LDS
    for (uint32_t i = tid; i < words; i += NT) bitmap[i] = 0u;
    if (tid < 2u) ctl[tid] = 0u;
    // a block's thread fetches one entry and its score of the student itself: ahead of the row, which the score is read behind
    static_assert(NT <= 64 || NT >= DDT_MAX_TOP, "an entry per thread");
    int32_t my_id = -1;
    float my_t = 0.f, my_x = 0.f;
    if (NT > 64 && tid < a.k) my_id = a.ids[row * a.teacher_stride + tid], my_t = a.values[row * a.teacher_stride + tid];
    HeldPack<T> raw[P > 0 ? P : 1];
    uint32_t own = tid;  // the thread's first pack; opaque, so that the packs' indexes and addresses are computed where they are used
    forget(own);
#pragma unroll
    for (int i = 0; i < P; ++i) raw[i].load(in, (own + (uint32_t)i * NT) * N, a.K);
    sync();
    auto enter = [&](uint32_t j, int32_t id, float t) {
      en.id[j] = id, en.t[j] = t;
      if (id >= 0) {
        ctl[0] = 1u;
        if (atomicOr(&bitmap[id >> 5], 1u << (id & 31)) >> (id & 31) & 1u) ctl[1] = 1u;
      }
    };
    if (NT > 64) {
      if ((uint32_t)my_id >= a.K) my_id = -1;
      if (tid < a.k) enter(tid, my_id, my_t);
      if (my_id >= 0) my_x = (float)in[my_id];
    } else {
      for (uint32_t j = tid; j < a.k; j += NT) {
        int32_t id = a.ids[row * a.teacher_stride + j];
        if ((uint32_t)id >= a.K) id = -1;
        enter(j, id, a.values[row * a.teacher_stride + j]);
        if (id >= 0) en.x[j] = (float)in[id];
      }
    }
    sync();
    if (ctl[0] == 0u) {  // no entry: nothing to learn from this row
      if (tid == 0u && a.loss) a.loss[row] = 0.f;
      if (GRAD) {
        const float zero[N] = {};
        for (uint32_t p = tid; p < packs; p += NT) store_pack(out, p * N, a.K, zero);
      }
      continue;
    }
    if (ctl[1]) {  // mark the entries whose class stands in front of them already
      for (uint32_t j0 = 0; j0 < a.k; j0 += NT) {
        const uint32_t j = j0 + tid;
        bool again = false;
        if (j < a.k && en.id[j] >= 0)
          for (uint32_t i = 0; i < j; ++i) again |= (en.id[i] & ~kAgain) == en.id[j];
        sync();
        if (again) en.id[j] |= kAgain;
        sync();
      }
    }
    typedef std::conditional_t<P == 0, double, float> Sum;
    RunSum<Sum> run(c2);
    uint32_t holds = 0u;  // packs (of the registers) that hold a listed class
    if (P > 0) {
      constexpr int C = P < 4 ? P : 4;  // packs that are summed at a time
#pragma unroll
      for (int i = 0; i < P; i += C) {
        forget(own);
        float x[(P > 0 ? C : 1) * N];
#pragma unroll
        for (int u = 0; u < C; ++u) {
          const uint32_t p = own + (uint32_t)(i + u) * NT, bits = p < packs ? listed_bits(p) : 0u;
          if (bits) holds |= 1u << (i + u), raw[i + u].clear(bits);
          float v[N];
          raw[i + u].get(v);
#pragma unroll
          for (uint32_t j = 0; j < N; ++j) x[u * N + j] = v[j];
        }
        if (own + (uint32_t)i * NT < packs) run.add(x, c2);
#pragma unroll
        for (int u = 0; u < C; ++u) raw[i + u].hold();
      }
    } else {
      uint32_t p0 = 0;
      for (; (p0 + 4u * NT) * N <= a.K; p0 += 4u * NT) {  // four packs of a thread in flight
        float x[4 * N];
        load_packs<T, NT>(in, p0 + tid, x);
#pragma unroll
        for (uint32_t u = 0; u < 4; ++u) {
          const uint32_t bits = listed_bits(p0 + tid + u * NT);
          if (bits) {
#pragma unroll
            for (uint32_t i = 0; i < N; ++i) x[u * N + i] = (bits >> i) & 1u ? -kInf : x[u * N + i];
          }
        }
        run.add(x, c2);
      }
      for (uint32_t p = p0 + tid; p < packs; p += NT) {
        float x[N];
        load_pack(in, p * N, a.K, -kInf, x);
        const uint32_t bits = listed_bits(p);
#pragma unroll
        for (uint32_t i = 0; i < N; ++i) x[i] = (bits >> i) & 1u ? -kInf : x[i];
        run.add(x, c2);
      }
    }
    ExpSum o = run.template finish<NT < 64 ? NT : 64>(c2, [&](float M) {
      Sum t = 0;
      for (uint32_t p = tid; p < packs; p += NT) {
        float x[N];
        load_pack(in, p * N, a.K, -kInf, x);
        const uint32_t bits = listed_bits(p);
        t += (Sum)sum_of<N>([&](uint32_t i) { return (bits >> i) & 1u ? 0.f : exp2_fast((x[i] - M) * c2); });
      }
      return (float)t;
    });
    if (NT > 64 && tid < a.k) en.x[tid] = my_x;
    if (NT > 64) {
      if (lane == 0u) part[2 * (tid >> 6)] = o.m, part[2 * (tid >> 6) + 1] = o.s;
      sync();
    }
    if (tid < 64u) {
      if (NT > 64) {
        o.m = lane < kWaves ? part[2 * lane] : -FLT_MAX, o.s = lane < kWaves ? part[2 * lane + 1] : 0.f;
        o.reduce_wave(c2);
      }
      const RowGrad g = row_loss<T, (NT < 64 ? NT : 64), GRAD>(a, row, en, bitmap, lane, o);
      if (GRAD && lane == 0u) ctl[2] = __float_as_uint(g.m), ctl[3] = __float_as_uint(g.coef);
    }
    if (GRAD) {
      sync();
      const float m = __uint_as_float(ctl[2]), coef = __uint_as_float(ctl[3]);
      auto write = [&](uint32_t p, const float (&x)[N], bool check) {
        const uint32_t bits = check ? listed_bits(p) : 0u;
        if (bits) {  // the listed classes of this pack are written already
#pragma unroll
          for (uint32_t i = 0; i < N; ++i)
            if (p * N + i < a.K && !((bits >> i) & 1u)) out[p * N + i] = (T)x[i];
        } else if (a.past_caches) {
          store_pack<T, true>(out, p * N, a.K, x);
        } else {
          store_pack<T>(out, p * N, a.K, x);
        }
      };
      // Two-byte gradients: coef goes into the exponent, with its sign put on afterwards -- two instructions per score less.  Its
      // rounding there is below 2^-16 for |m c| up to 256, next to a result that is rounded to 11 bits at most.
      const float b = log2f(fabsf(coef)) - m * c2;
      const uint32_t sign = __float_as_uint(coef) & 0x80000000u;
      const bool folded = sizeof(T) == 2 && fabsf(m * c2) <= 256.f;
      auto plain = [&](float x) { return coef * exp2_fast((x - m) * c2); };
      auto in_exponent = [&](float x) { return __uint_as_float(__float_as_uint(exp2_fast(fmaf(x, c2, b))) ^ sign); };
      if (P > 0 && (sizeof(T) == 4 || folded)) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
          forget(own);
          if (own + (uint32_t)i * NT < packs) {
            float x[N];
            raw[i].get(x);
#pragma unroll
            for (uint32_t j = 0; j < N; ++j) x[j] = sizeof(T) == 4 ? plain(x[j]) : in_exponent(x[j]);
            write(own + (uint32_t)i * NT, x, (holds >> i) & 1u);
          }
        }
      } else {
        // from the row's end, which was read last and is the likeliest to be in the L2 still; four packs of a thread in flight
        const uint32_t whole = P == 0 && (sizeof(T) == 4 || folded) ? a.K / (4u * NT * N) * (4u * NT) : 0u;
        if (P == 0)
          for (uint32_t p0 = whole; p0 > 0u;) {
            p0 -= 4u * NT;
            float x[4 * N];
            load_packs<T, NT>(in, p0 + tid, x);
#pragma unroll
            for (uint32_t u = 0; u < 4; ++u) {
              float y[N];
#pragma unroll
              for (uint32_t j = 0; j < N; ++j) y[j] = sizeof(T) == 4 ? plain(x[u * N + j]) : in_exponent(x[u * N + j]);
              write(p0 + tid + u * NT, y, true);
            }
          }
        for (uint32_t p = whole + tid; p < packs; p += NT) {
          float x[N];
          load_pack(in, p * N, a.K, -kInf, x);
#pragma unroll
          for (uint32_t j = 0; j < N; ++j) x[j] = plain(x[j]);
          write(p, x, true);
        }
      }
    }
  }
}

// up to 32 classes: a thread per row, rows staged in LDS and their gradients collected there in fp32.  1 M x 10 fp32, k = 4: 47 us, 1150
// vector instructions per wave of 64 rows (30 us' worth of issue): the 64-bit numbers of the rows bound it, not the 120 MB.  KK > 0:
// k = KK entries per row, in registers with their exponentials; KK = 0: any number, read and computed again where they are needed.
// (Up to KK = 5, 124 registers and four waves per SIMD; without the branches on entries it is 135 and 52 -> 56 us.)
// (KK = 2 is held to the 96 registers of five waves: a register more cost 1 M x 10 bf16 39 -> 42 us.)
template <class T, int KK, bool GRAD>
__global__ __launch_bounds__(256, KK == 2 ? 5 : 1) void distill_thread_kernel(const DistillArgs a) {
  T* stage = reinterpret_cast<T*>(lds_words);
  const uint32_t pitch = staged_pitch<T>(a.K), gpitch = a.K | 1u;
  float* gstage = reinterpret_cast<float*>(lds_words + (256u * pitch * sizeof(T)) / 4u);
  constexpr double kLn2 = 0.69314718055994530942;
  const float c2 = a.scale;
  const double inv_T = a.inv_T, x_scale = (double)c2;
  for (uint64_t r0 = (uint64_t)blockIdx.x * 256u; r0 < a.n; r0 += (uint64_t)gridDim.x * 256u) {
    const uint32_t rows = (uint32_t)(a.n - r0 < 256u ? a.n - r0 : 256u);
    const uint32_t tid = forgotten(threadIdx.x);
    const bool active = tid < rows;
    const uint64_t row = r0 + tid;
    const int32_t* ids = a.ids + row * a.teacher_stride;
    const float* tv = a.values + row * a.teacher_stride;
    int32_t id[KK > 0 ? KK : 1];
    float t[KK > 0 ? KK : 1];
    double eq[KK > 0 ? KK : 1][2];
    float given_lse = 0.f, weight = 1.f;
    if (active) {
      if (KK > 0) __builtin_memcpy(id, ids, sizeof(id)), __builtin_memcpy(t, tv, sizeof(t));
      if (a.lse) given_lse = a.lse[row];
      if (GRAD && a.weight) weight = a.weight[row * a.weight_stride];
    }
    __syncthreads();
    stage_rows(static_cast<const T*>(a.in), r0, rows, a.K, a.stride, stage, pitch);
    __syncthreads();
    if (active) {
      const T* x = stage + tid * pitch;
      float* g = gstage + tid * gpitch;
      auto each = [&](auto f) {  // f(entry, class, score) of the row's entries, in order
        if constexpr (KK > 0) {
#pragma unroll
          for (int j = 0; j < KK; ++j)
            if ((uint32_t)id[j] < a.K) f(j, (uint32_t)id[j], t[j]);
        } else {
          for (uint32_t j = 0; j < a.k; ++j)
            if ((uint32_t)ids[j] < a.K) f(j, (uint32_t)ids[j], tv[j]);
        }
      };
      uint32_t listed = 0u, entries = 0u;
      float tm = -FLT_MAX;
      each([&](uint32_t, uint32_t c, float v) { listed |= 1u << c, tm = fmaxf(tm, v), ++entries; });
      if (listed == 0u) {
        if (a.loss) a.loss[row] = 0.f;
        if (GRAD)
          for (uint32_t c = 0; c < a.K; ++c) g[c] = 0.f;
      } else {
        float om = -FLT_MAX, sm = -FLT_MAX, os = 0.f;
#pragma unroll 4
        for (uint32_t c = 0; c < a.K; ++c) {
          const float v = (float)x[c];
          const bool on = (listed >> c) & 1u;
          sm = fmaxf(sm, on ? v : sm), om = fmaxf(om, on ? om : v);
        }
#pragma unroll 4
        for (uint32_t c = 0; c < a.K; ++c) {
          const float e = exp2_fast(((float)x[c] - om) * c2);
          os += (listed >> c) & 1u ? 0.f : e;
          if (GRAD) g[c] = e;  // (what stands there for a listed class is written over)
        }
        const float M = fmaxf(om, sm);
        const double shift = a.lse ? (double)given_lse : (double)tm * inv_T;
        auto student = [&](uint32_t c) { return ((double)(float)x[c] - (double)M) * x_scale; };
        auto teacher = [&](float v) { return exp2_64(((double)v * inv_T - shift) * kLog2e); };
        double zs = 0.0, ts = 0.0;
        uint32_t open = listed;  // classes of the list that are still to come
        each([&](uint32_t j, uint32_t c, float v) {
          const double e = exp2_64(student(c)), q = teacher(v);
          if (KK > 0) eq[KK > 0 ? j : 0][0] = e, eq[KK > 0 ? j : 0][1] = q;
          zs += (open >> c) & 1u ? e : 0.0;
          ts += q;
          open &= ~(1u << c);
        });
        const double far = exp2_64(((double)om - (double)M) * x_scale), Z = (double)os * far + zs, log_Z = log_64(Z);
        const double log_T = a.lse ? shift : shift + log_64(ts), scale = a.lse ? 1.0 : inverse_64(ts);
        double Q = a.lse ? ts : ts * scale, rest_s = 0.0, loss = 0.0;
        if (a.lse && os > 0.f && Q < 1.0) {
          rest_s = (1.0 - Q) * inverse_64((double)os);
          loss = (1.0 - Q) * (log_64(rest_s) - (((double)om - (double)M) * x_scale * kLn2 - log_Z));
          Q = 1.0;
        } else if (a.lse && os == 0.f && (uint32_t)__popc(listed) < a.K && rest_counts(Q, (float)shift)) {
          loss = __builtin_inf();
        }
        const bool none = !(Z > 0.0 && Q >= 0.0 && Q < __builtin_inf());  // (as in row_loss)
        const double w = (double)weight * inv_T, p_scale = none ? __builtin_nan("") : Q * inverse_64(Z);
        if (GRAD) {
          const float coef = os == 0.f && !none ? 0.f : (float)((p_scale * far - rest_s) * w);
#pragma unroll 4
          for (uint32_t c = 0; c < a.K; ++c) g[c] *= coef;
        }
        const bool repeats = entries != (uint32_t)__popc(listed);
        open = listed;
        each([&](uint32_t j, uint32_t c, float v) {
          const double q = KK > 0 ? eq[KK > 0 ? j : 0][1] : teacher(v);
          if (!(q == 0.0)) loss += q * scale * (((double)v * inv_T - log_T) - (student(c) * kLn2 - log_Z));
          if (GRAD && ((open >> c) & 1u)) {
            open &= ~(1u << c);
            double qc = q;
            if (repeats)  // further entries of this class, in their order
              for (uint32_t i = j + 1u; i < a.k; ++i)
                if (ids[i] == (int32_t)c) qc += teacher(tv[i]);
            g[c] = (float)(((KK > 0 ? eq[KK > 0 ? j : 0][0] : exp2_64(student(c))) * p_scale - qc * scale) * w);
          }
        });
        if (a.loss) a.loss[row] = none ? __builtin_nanf("") : (float)loss;
      }
    }
    if (GRAD) {
      __syncthreads();
      T* out = static_cast<T*>(a.grad);
      if (a.grad_stride == a.K && a.K > 1u) {
        constexpr uint32_t N = Pack<T>::N;
        const uint32_t total = rows * a.K, magic = (uint32_t)((0x100000000ull + a.K - 1u) / a.K);
        T* dst = out + r0 * a.K;
        for (uint32_t i = tid * N; i < total; i += 256u * N) {
          uint32_t r = __umulhi(i, magic), c = i - r * a.K;
          float v[N];
#pragma unroll
          for (uint32_t j = 0; j < N; ++j) {
            v[j] = i + j < total ? gstage[r * gpitch + c] : 0.f;
            if (++c == a.K) c = 0u, ++r;
          }
          if (a.past_caches) store_pack<T, true>(dst, i, total, v);
          else store_pack<T>(dst, i, total, v);
        }
      } else {
        for (uint32_t r = tid >> 5; r < rows; r += 8u)
          for (uint32_t c = tid & 31u; c < a.K; c += 32u) out[(r0 + r) * a.grad_stride + c] = (T)gstage[r * gpitch + c];
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------------------------------
template <class Kern, class... Args>
hipError_t launch(Kern kern, uint64_t blocks, uint32_t threads, uint32_t lds, hipStream_t s, const Args&... args) {
  (void)hipGetLastError();  // do not inherit a stale error
  if (lds > 64u * 1024u) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  constexpr uint64_t kMaxBlocks = 1u << 20;  // every kernel strides over the rest
  hipLaunchKernelGGL(kern, dim3((uint32_t)(blocks < kMaxBlocks ? blocks : kMaxBlocks)), dim3(threads), lds, s, args...);
  return hipGetLastError();
}

template <class T>
hipError_t adjust_typed(const AdjustArgs& a, bool class_major, hipStream_t s) {
  constexpr uint32_t N = Pack<T>::N;
  AdjustTiles t{};
  if (class_major) {
    // Without a history a tile is 256 packs of rows times 16 classes (300,000 x 100 fp32 41 us; 4 classes 42, 64 classes 73, 64 packs 43;
    // 20,000 x 2000 71, 58, 79, 59).  The counters of a history are 64 rows times 256 classes, 64 KB (64 x 64, us: 300,000 x 100 with 13
    // entries a row 205 -> 274, 100,000 x 300 with 40 454 -> 262, 20,000 x 2000 with 200 382 -> 338).
    t.rows = a.history ? 64u : 256u * N;
    t.classes = a.K < (a.history ? 256u : 16u) ? a.K : (a.history ? 256u : 16u);
    t.class_tiles = (a.K + t.classes - 1) / t.classes;
    t.tiles = (a.n + t.rows - 1) / t.rows * t.class_tiles;
    if (a.history) return launch(adjust_classes_kernel<T, true>, t.tiles, 256, t.rows * t.classes * 4u, s, a, t);
    return launch(adjust_classes_kernel<T, false>, t.tiles, 256, 0, s, a, t);
  }
  const uint64_t row_packs = (a.K + N - 1) / N;
  // 512 packs per tile, 256 if that leaves too few tiles for the chip (64 x 128000 bf16, 100 / 8192 entries of history: 14 / 21 us, with
  // 1024 packs 17 / 24; 256 packs with 100 / 2000 entries 14.7 / 15.8, 512 packs 13.2 / 14.9; below 2^17 packs both are the call's 12 us).
  // Every tile of a row reads the row's whole history: from 6000 entries a row on, 1024 threads share that and 1024 packs (32 x 50257 fp32
  // with 15,000 / 50,000 entries a row: 14.0 / 20.8 us, with 256 threads 14.9 / 34.2; 64 x 128000 bf16 with 6000 / 15,000: 26.7 / 28.9,
  // 19.5 / 27.3).
  const bool small = a.n * row_packs < (1u << 17), many = a.history && a.history_len / a.n > 6000u;
  const uint32_t budget = many ? 1024u : small ? 256u : 512u;
  const uint32_t ppr = (uint32_t)(row_packs < budget ? row_packs : budget);
  t.classes = ppr * N;
  t.rows = budget / ppr;
  t.magic = ppr > 1u ? (uint32_t)((0x100000000ull + ppr - 1u) / ppr) : 0u;
  t.class_tiles = (row_packs + ppr - 1) / ppr;
  t.tiles = (a.n + t.rows - 1) / t.rows * t.class_tiles;
  const uint32_t lds = a.history ? t.rows * t.classes * 4u : 0u;
  if (many) return launch(adjust_rows_kernel<T, true, 1024, 1>, t.tiles, 1024, lds, s, a, t);
  if (a.history) return small ? launch(adjust_rows_kernel<T, true, 256, 1>, t.tiles, 256, lds, s, a, t)
                              : launch(adjust_rows_kernel<T, true, 256, 2>, t.tiles, 256, lds, s, a, t);
  return small ? launch(adjust_rows_kernel<T, false, 256, 1>, t.tiles, 256, lds, s, a, t)
               : launch(adjust_rows_kernel<T, false, 256, 2>, t.tiles, 256, lds, s, a, t);
}

template <class T, bool CM>
hipError_t top_thread(const TopArgs& a, hipStream_t s) {
  const uint64_t blocks = (a.n + 255) / 256;
  const uint32_t lds = CM ? 0u : 256u * (uint32_t)sizeof(T) * ((((a.K + 4 / sizeof(T) - 1) / (4 / sizeof(T))) | 1u) * (uint32_t)(4 / sizeof(T)));
  switch (a.k) {
    case 1: return launch(top_thread_kernel<T, CM, 1>, blocks, 256, lds, s, a);
    case 2: return launch(top_thread_kernel<T, CM, 2>, blocks, 256, lds, s, a);
    case 3: return launch(top_thread_kernel<T, CM, 3>, blocks, 256, lds, s, a);
    case 4: return launch(top_thread_kernel<T, CM, 4>, blocks, 256, lds, s, a);
    case 5: return launch(top_thread_kernel<T, CM, 5>, blocks, 256, lds, s, a);
    case 6: return launch(top_thread_kernel<T, CM, 6>, blocks, 256, lds, s, a);
    case 7: return launch(top_thread_kernel<T, CM, 7>, blocks, 256, lds, s, a);
    default: return launch(top_thread_kernel<T, CM, 8>, blocks, 256, lds, s, a);
  }
}
template <class T, bool CM>
hipError_t top_wave(const TopArgs& a, hipStream_t s) {
  constexpr uint32_t N = Pack<T>::N, rows = top_wave_rows(CM), threads = top_wave_waves(CM) * 64u;
  const uint64_t blocks = (a.n + rows - 1) / rows;
  const uint32_t lds = top_wave_waves(CM) * wave_list(a.k) * 8u + (CM ? a.K * kStagePitch * 4u : 0u), packs = (a.K + N - 1) / N;
  if (packs <= 64u) return launch(top_wave_kernel<T, CM, 1>, blocks, threads, lds, s, a);
  if (packs <= 128u) return launch(top_wave_kernel<T, CM, 2>, blocks, threads, lds, s, a);
  if (packs <= 256u) return launch(top_wave_kernel<T, CM, 4>, blocks, threads, lds, s, a);
  if constexpr (N == 4) return launch(top_wave_kernel<T, CM, 8>, blocks, threads, lds, s, a);
  return hipErrorInvalidValue;
}
template <class T, int NT>
hipError_t top_block(const TopArgs& a, hipStream_t s) {
  return launch(top_block_kernel<T, NT>, a.n, NT, 4u * top_block_words(NT), s, a);
}
template <class T, bool CM>
hipError_t top_rank(const TopArgs& a, hipStream_t s) {
  constexpr uint32_t per_word = 4 / sizeof(T);
  const uint32_t staged = CM ? 0u : 256u * (uint32_t)sizeof(T) * ((((a.K + per_word - 1) / per_word) | 1u) * per_word);
  const uint32_t out = 256u * 8u * ((a.k < a.K ? a.k : a.K) | 1u), lds = staged > out ? staged : out;
  const uint64_t blocks = (a.n + 255) / 256;
  return a.K <= 16u ? launch(top_rank_kernel<T, CM, 16>, blocks, 256, lds, s, a) : launch(top_rank_kernel<T, CM, 32>, blocks, 256, lds, s, a);
}
template <class T, bool CM>
hipError_t top_lanes(const TopArgs& a, uint32_t p, hipStream_t s) {
  const uint64_t blocks = (a.n + 15) / 16;
  const uint32_t lds = CM ? a.K * kStagePitch * 4u : 0u;
  if (p == 1u) return launch(top_lanes_kernel<T, CM, 1>, blocks, 256, lds, s, a);
  if (p == 2u) return launch(top_lanes_kernel<T, CM, 2>, blocks, 256, lds, s, a);
  if (p == 4u) return launch(top_lanes_kernel<T, CM, 4>, blocks, 256, lds, s, a);
  if constexpr (Pack<T>::N == 4) return launch(top_lanes_kernel<T, CM, 8>, blocks, 256, lds, s, a);
  return hipErrorInvalidValue;
}
template <class T>
hipError_t top_typed(const TopArgs& a, bool class_major, hipStream_t s) {
  constexpr uint32_t N = Pack<T>::N;
  // counted ranks against 16 lanes or a wave per row, us: 1 M x 16, k = 9 42 / 218, 1 M x 32, k = 17 152 / 1274 (4096 x 32 15 / 11)
  if (a.K <= 32u && a.k > 8u) return class_major ? top_rank<T, true>(a, s) : top_rank<T, false>(a, s);
  // A thread per row reads class-major rows as they lie; with many classes it takes many rows to fill the chip.  Against 16 lanes or a wave,
  // us, k = 4, class-major fp32: 32,768 x 40 / 300 10.4 / 52 against 10.7 / 27, 65,536 x 40 / 300 / 1000 10.6 / 51 / 152 against 12.6 / 42 /
  // 125, 131,072 x 300 59 against 73, 300,000 x 100 34 against 58.  Row-major: 32,768 x 64 17.9 against 10.6, 65,536 x 40 11.7 against 11.7,
  // 1 M x 40 81 against 126, 1 M x 64 fp32 / bf16 164 / 87 against 124 / 161, 1 M x 10 (k = 3) 18 against 104.
  if (class_major && a.k <= 8u && (a.K <= 32u || a.n >= 65536u)) return top_thread<T, true>(a, s);
  if (!class_major && a.k <= 8u && (a.K <= 32u || (a.K <= 64u && a.n >= 65536u))) return top_thread<T, false>(a, s);
  if (class_major && a.K > kTopMaxClassMajor) return hipErrorInvalidValue;
  // 16 lanes per row take out the best k times, 5 instructions per score and 40 each: against about 600 per row for a whole wave.  (us, fp32,
  // 16 lanes / wave: 75,000 x 200, k = 8 / 12 / 16 38 / 51 / 65 against 52 / 53 / 53, 30,000 x 500, k = 8 / 12 / 16 32 / 42 / 52 against 27 /
  // 28 / 29, 150,000 x 100, k = 16 75 against 94, 16,384 x 500, k = 4 14 against 17; 4096 rows and fewer are the call's 11 us either way.)
  const uint32_t packs = (a.K + N - 1) / N, p = packs <= 16u ? 1u : packs <= 32u ? 2u : packs <= 64u ? 4u : 8u;
  if (a.n >= 4096u && a.k <= 16u && packs <= 512u / N && a.k * (5u * p * N + 40u) <= 2400u)
    return class_major ? top_lanes<T, true>(a, p, s) : top_lanes<T, false>(a, p, s);
  if (class_major) return top_wave<T, true>(a, s);
  // a wave against a block of 256, us: 16,384 x 1000 fp32, k = 20 / 200 24 / 106 against 54 / 248, 16,384 x 2048 39 / 146 against 56 / 274,
  // 16 x 2048, k = 200 29 against 19
  if (a.K <= 2048u) return top_wave<T, false>(a, s);
  // 256 threads against 512 (1024 for up to 256 rows), us, k = 50: 4000 x 16,000 fp32 / bf16 60 / 35 against 67 / 47, 4000 x 24,000 80 / 47
  // against 87 / 63, 1000 x 50,000 41 / 24 against 43 / 27, 200 x 50,000 17 / 13 against 14 / 12.  512 against 1024, bf16: 256 x 128,000 18
  // either way, 64 x 128,000 15.7 / 14.7, 384 x 50,257 16 / 21, 1024 x 128,000 58 / 66
  if (a.K <= 16384u) return top_block<T, 256>(a, s);
  return a.n > 256u ? top_block<T, 512>(a, s) : top_block<T, 1024>(a, s);
}

template <class T, int NT, int P, bool GRAD>
hipError_t distill_rows(const DistillArgs& a, hipStream_t s) {
  constexpr uint32_t groups = NT < 256 ? 256u / NT : 1u;
  const uint32_t lds = groups * 4u * distill_words(a.K, a.k, NT);
  return launch(distill_kernel<T, NT, P, GRAD>, (a.n + groups - 1) / groups, NT < 256 ? 256 : NT, lds, s, a);
}
template <class T, bool GRAD>
hipError_t distill_typed(const DistillArgs& a, hipStream_t s) {
  constexpr uint32_t per_word = 4 / sizeof(T);
  // a thread per row against 16 lanes, us, gradient: 1 M x 10 fp32, k = 2 / 8 37 / 105 against 285 / 305, 1 M x 32 128 / 213 against 308 / 334
  // (4096 x 32, k = 8 19 against 12); entries in registers against reading them again, 1 M x 10, k = 1 .. 5: 33 37 41 44 47 against 39 45 51 57 63
  if (a.K <= 32u) {
    const uint32_t pitch = (((a.K + per_word - 1) / per_word) | 1u) * per_word;
    const uint32_t lds = 256u * (pitch * (uint32_t)sizeof(T) + (GRAD ? (a.K | 1u) * 4u : 0u));
    const uint64_t blocks = (a.n + 255) / 256;
    switch (a.k) {
      case 1: return launch(distill_thread_kernel<T, 1, GRAD>, blocks, 256, lds, s, a);
      case 2: return launch(distill_thread_kernel<T, 2, GRAD>, blocks, 256, lds, s, a);
      case 3: return launch(distill_thread_kernel<T, 3, GRAD>, blocks, 256, lds, s, a);
      case 4: return launch(distill_thread_kernel<T, 4, GRAD>, blocks, 256, lds, s, a);
      case 5: return launch(distill_thread_kernel<T, 5, GRAD>, blocks, 256, lds, s, a);
      default: return launch(distill_thread_kernel<T, 0, GRAD>, blocks, 256, lds, s, a);
    }
  }
  const uint32_t packs = (a.K + Pack<T>::N - 1) / Pack<T>::N;
  // Short rows: what a row does once (its 64-bit numbers, its reductions) outweighs its scores, so four of them share a wave -- where there
  // are rows enough to fill the chip that way.  (100 M scores, us, 64 -> 16 threads per row: loss + gradient of 200 bf16 classes 922 -> 333,
  // 500 fp32 386 -> 271, 1500 bf16 212 -> 171; 1000 fp32 239 -> 258.  8192 x 400 fp32 18 -> 14, 4096 x 1000 15 -> 18.5, fewer rows are the
  // call's 12.5 either way; 50,000 x 300, k = 16 / 64 77 / 108 -> 43 / 105.)
  if (a.n >= 4096u && a.k <= 64u && packs <= 256u) {
    if (packs <= 16u) return distill_rows<T, 16, 1, GRAD>(a, s);
    if (packs <= 32u) return distill_rows<T, 16, 2, GRAD>(a, s);
    if (packs <= 64u) return distill_rows<T, 16, 4, GRAD>(a, s);
    if (packs <= 128u) return distill_rows<T, 16, 8, GRAD>(a, s);
    return distill_rows<T, 16, 16, GRAD>(a, s);
  }
  // a wave against a block of 256, gradient, us: 60,000 rows of 64 / 256 / 512 packs fp32 132 / 179 / 272 against 381 / 417 / 445, 600 rows of
  // 512 packs 15.3 against 12.8
  if (packs <= 64u) return distill_rows<T, 64, 1, GRAD>(a, s);
  if (packs <= 128u) return distill_rows<T, 64, 2, GRAD>(a, s);
  if (packs <= 256u) return distill_rows<T, 64, 4, GRAD>(a, s);
  if (packs <= 512u) return distill_rows<T, 64, 8, GRAD>(a, s);
  // few rows: as many threads on each as there are.  Else enough blocks per CU that one row's ends are hidden behind the other rows'
  // packs -- for the gradient no more than keep their rows in the 256 MB cache until their second read, and in registers where a thread's
  // packs fill them.  (us with 256 / 512 / 1024 threads: loss of 2048 x 50257 fp16 51 / 54 / 72; gradient of 8192 x 128000 bf16
  // 1123 / 951 / 1148, 2000 x 100000 fp32 457 / 402 / 400; 200 M bf16 scores with 512 / 1024 threads, rows of 5000 packs 213 / 333, of 16,000
  // 223 / 245, of 20,000 221 / 221.  1024 threads / fewer for few rows: gradient of 256 x 20,000 bf16 13.7 / 16.7, of 512 24.3 / 20.1, loss of
  // 256 x 50,257 10.9 / 12.5, of 512 17.9 / 14.3.)
  if (a.n <= 512u) return distill_rows<T, 1024, 0, GRAD>(a, s);
  // four packs a thread in registers against reading twice, us: 20,000 rows of 600 / 1000 packs, gradient fp32 162 / 179 against 187 / 228, bf16
  // 226 / 251 against 212 / 261, loss fp32 66 / 70 against 72 / 88
  if (packs <= 1024u) return distill_rows<T, 256, 4, GRAD>(a, s);
  if constexpr (GRAD) {
    // Reading twice against 16 packs a thread in registers (136 of them: three waves per SIMD, however many of the packs are there), us: 12,000
    // rows of 1100 / 2000 / 2900 / 3300 / 4000 packs fp32 115 / 192 / 268 / 290 / 360 against 193 / 221 / 252 / 268 / 304, of 2900 bf16 276
    // against 301; 1000 rows of 4000, which the cache holds, 33 against 38.
    if (packs <= 3000u) return distill_rows<T, 256, 0, GRAD>(a, s);
    if (packs <= 4096u) return distill_rows<T, 256, 16, GRAD>(a, s);
    return packs <= 16384u ? distill_rows<T, 512, 0, GRAD>(a, s) : distill_rows<T, 1024, 0, GRAD>(a, s);
  }
  return distill_rows<T, 256, 0, GRAD>(a, s);
}

}  // namespace

hipError_t launch_adjust(const AdjustArgs& a, uint32_t dtype, bool class_major, hipStream_t s) {
  if (a.n == 0) return hipSuccess;
  if (dtype == DDT_FP32) return adjust_typed<float>(a, class_major, s);
  return dtype == DDT_FP16 ? adjust_typed<_Float16>(a, class_major, s) : adjust_typed<__bf16>(a, class_major, s);
}
hipError_t launch_top(const TopArgs& a, uint32_t dtype, bool class_major, hipStream_t s) {
  if (a.n == 0) return hipSuccess;
  if (dtype == DDT_FP32) return top_typed<float>(a, class_major, s);
  return dtype == DDT_FP16 ? top_typed<_Float16>(a, class_major, s) : top_typed<__bf16>(a, class_major, s);
}
hipError_t launch_distill(const DistillArgs& args, uint32_t dtype, hipStream_t s) {
  if (args.n == 0) return hipSuccess;
  // student and gradient do not both fit the 256 MB cache: the gradient goes past it (8192 x 128000 bf16 1057 -> 963 us)
  DistillArgs a = args;
  a.past_caches = a.n * a.K * (dtype == DDT_FP32 ? 4u : 2u) > (128ull << 20);
  if (dtype == DDT_FP32) return a.grad ? distill_typed<float, true>(a, s) : distill_typed<float, false>(a, s);
  if (dtype == DDT_FP16) return a.grad ? distill_typed<_Float16, true>(a, s) : distill_typed<_Float16, false>(a, s);
  return a.grad ? distill_typed<__bf16, true>(a, s) : distill_typed<__bf16, false>(a, s);
}

}  // namespace ddt
