// Log probabilities of given tokens with the distribution's entropy, its largest
// alternatives, and the gradient (gfx950).  For a row x of V logits with the
// largest m, a_j = (x_j - m) log2(e), s = sum_j 2^a_j, t = sum_j a_j 2^a_j:
//
//   log p_j = (x_j - m) - ln 2 log2 s  (in fp64),
//   H = -sum_j p_j log p_j = ln 2 (log2 s - t / s)
//   d/dx_j  (a log p_i + h H + sum_k b_k log p_{i_k})
//         = a [j = i] + sum_k b_k [j = i_k] - p_j (a + sum_k b_k + h (log p_j + H))
//
// The maximum is taken off in the logits' own unit: the difference is exact near
// it and 0 at it, whatever the logits' size.  (One fma, x_j log2(e) + n with n =
// -m log2(e) rounded, would save an instruction a logit, but carries n's rounding
// into every exponent: up to 64 at m = 1e9, and at the type's lowest value n itself
// is infinite, so that a mask of a large finite value over a whole piece made
// its row NaN.  8192 x 32000 bf16: 86 us so, 91 now; 20 alternatives 122 and 126;
// forward and gradient 282 and 284.)
//
// All sums in fp32.  Both directions are bound by the bytes of the logits: the
// forward reads them once, the backward reads them and writes the gradient.
//
// Forward: one workgroup a row, which stands in registers (64 logits a thread)
// while its maximum, then the sums, then the alternatives are taken, so that no
// running maximum rescales sums inside a piece; longer rows go in pieces joined
// by their maxima.  bf16 logits stay packed and are widened anew in each
// pass (the registers are made opaque in between, or the compiler keeps all 64
// widened: 8192 x 32000 with 20 alternatives 176 us, against 126; without
// alternatives level, 91).
//
// Alternatives, k of them in the order of (value, lowest index first).  Among
// the 64 maxima of 64 disjoint groups of the piece's logits the k-th largest,
// T, is at most the k-th largest logit; logits from T up, some 1.2 k on average,
// go to a list in LDS.  A list that overflows (values sorted against the groups,
// many ties) has T replaced by the piece's exact k-th value, by its digits, and
// ties at it, as those at -inf where the row has fewer than k others, in the
// order of their index.  A candidate's place is the number of larger ones.
#include "common.h"
#include "prof.h"

namespace sa {
namespace {

constexpr int kMaxTop = 64;
constexpr int kList = 512;   // candidates of a piece
// 2^a is 0 in fp32 from here down: a logit of -inf is taken as this in a 2^a,
// which is then 0 and stays so under any factor
constexpr float kFloor = -160.0f;
constexpr double kLn2 = 0.6931471805599453;

constexpr uint32_t kOrderNan = 0xffffffffu, kOrderInf = 0xff800000u, kOrderLow = 0x007fffffu;   // NaN, +inf, -inf
// floats in the order of their values as unsigned numbers above 0: -inf lowest,
// NaN highest, both zeros the same
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return x != x ? kOrderNan : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return o == kOrderNan ? __builtin_nanf("") : __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}

// A row is read through a buffer resource that starts at the 16-byte boundary
// at or below it (`off` logits before it) and ends with it: reads behind the
// end return 0 in hardware, and octets that are not all the row's get -inf in
// those places.
struct Raw8f {
  float4 a, b;
};
template <typename T>
__device__ __forceinline__ __amdgpu_buffer_rsrc_t row_rsrc(const T* x, int off, int V) {
  const int bytes = static_cast<int>(((off + static_cast<long>(V)) * sizeof(T) + 3) & ~3l);
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(x - off), static_cast<short>(0), bytes, 0x00020000);
}
// the octet at j0 (j0 + off a multiple of 8), j0 < V or not
__device__ __forceinline__ void load8(__amdgpu_buffer_rsrc_t r, int j0, int off, uint4& raw) {
  raw = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, (j0 + off) * 2, 0, 0));
}
__device__ __forceinline__ void load8(__amdgpu_buffer_rsrc_t r, int j0, int off, Raw8f& raw) {
  const int at = (j0 + off) * 4;
  raw.a = __builtin_bit_cast(float4, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0));
  raw.b = __builtin_bit_cast(float4, __builtin_amdgcn_raw_buffer_load_b128(r, at + 16, 0, 0));
}
__device__ __forceinline__ void edge8(int j0, int V, uint4& raw) {
  if (j0 >= 0 && j0 + 8 <= V) return;
  uint32_t u[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (j0 + i < 0 || j0 + i >= V)
      u[i >> 1] = (i & 1) ? (u[i >> 1] & 0xffffu) | 0xff800000u : (u[i >> 1] & 0xffff0000u) | 0xff80u;
  raw = uint4{u[0], u[1], u[2], u[3]};
}
__device__ __forceinline__ void edge8(int j0, int V, Raw8f& raw) {
  if (j0 >= 0 && j0 + 8 <= V) return;
  float u[8] = {raw.a.x, raw.a.y, raw.a.z, raw.a.w, raw.b.x, raw.b.y, raw.b.z, raw.b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (j0 + i < 0 || j0 + i >= V) u[i] = -__builtin_huge_valf();
  raw.a = make_float4(u[0], u[1], u[2], u[3]);
  raw.b = make_float4(u[4], u[5], u[6], u[7]);
}
__device__ __forceinline__ float elem(const uint4& r, int i) {
  const uint32_t w = (i >> 1) == 0 ? r.x : (i >> 1) == 1 ? r.y : (i >> 1) == 2 ? r.z : r.w;
  return (i & 1) ? bf16hi_to_f32(w) : bf16lo_to_f32(w);
}
__device__ __forceinline__ float elem(const Raw8f& r, int i) {
  const float4& q = i < 4 ? r.a : r.b;
  return (i & 3) == 0 ? q.x : (i & 3) == 1 ? q.y : (i & 3) == 2 ? q.z : q.w;
}
// the same at a place known at run time
__device__ __forceinline__ float pick(const uint4& r, int i) {
  const uint32_t a = (i & 2) ? r.y : r.x, b = (i & 2) ? r.w : r.z, w = (i & 4) ? b : a;
  return __uint_as_float((i & 1) ? w & 0xffff0000u : w << 16);
}
__device__ __forceinline__ float pick(const Raw8f& r, int i) {
  const float a = (i & 1) ? r.a.y : r.a.x, b = (i & 1) ? r.a.w : r.a.z;
  const float c = (i & 1) ? r.b.y : r.b.x, d = (i & 1) ? r.b.w : r.b.z;
  return (i & 4) ? ((i & 2) ? d : c) : ((i & 2) ? b : a);
}
template <typename T> struct RawOf;
template <> struct RawOf<bf16> { using type = uint4; };
template <> struct RawOf<float> { using type = Raw8f; };

// the compiler may not carry values derived from these registers past this point
__device__ __forceinline__ void opaque(uint4& r) { asm volatile("" : "+v"(r.x), "+v"(r.y), "+v"(r.z), "+v"(r.w)); }
__device__ __forceinline__ void opaque(Raw8f& r) {
  asm volatile("" : "+v"(r.a.x), "+v"(r.a.y), "+v"(r.a.z), "+v"(r.a.w), "+v"(r.b.x), "+v"(r.b.y), "+v"(r.b.z), "+v"(r.b.w));
}

__device__ __forceinline__ float max8(const uint4& r, float m) {
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) m = fmaxf(fmaxf(m, bf16lo_to_f32(w[i])), bf16hi_to_f32(w[i]));
  return m;
}
__device__ __forceinline__ float max8(const Raw8f& r, float m) {
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, elem(r, i));
  return m;
}

// over the workgroup, the same order of sums whatever the launch
template <int NW>
__device__ __forceinline__ float block_max(float v, float* red) {
  v = wave_max(v);
  if constexpr (NW > 1) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) v = fmaxf(v, red[i]);
  }
  return v;
}
template <int NW>
__device__ __forceinline__ void block_sum2(float& u, float& v, float2* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    u += __shfl_xor(u, o, 64);
    v += __shfl_xor(v, o, 64);
  }
  if constexpr (NW > 1) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_float2(u, v);
    __syncthreads();
    u = v = 0.0f;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      u += red[i].x;
      v += red[i].y;
    }
  }
}

// exclusive count over the workgroup's threads of c, and the total
template <int NW>
__device__ __forceinline__ int block_scan(int c, int* wtot, int& total) {
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6;
  int incl = c;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int t = __shfl_up(incl, o, 64);
    if (lane >= o) incl += t;
  }
  __syncthreads();
  if (lane == 63) wtot[wid] = incl;
  __syncthreads();
  int pre = incl - c;
  total = 0;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    pre += i < wid ? wtot[i] : 0;
    total += wtot[i];
  }
  return pre;
}

// sums s, t of two sets of logits against their maxima m (-inf: no finite logit,
// s and t are 0 or NaN), joined against the larger one.  No sum is infinite, as
// 2^a <= 1, so a factor of 0 leaves 0 or the NaN.
__device__ __forceinline__ void join_sums(float& m, float& s, float& t, float m2, float s2, float t2) {
  const float mm = fmaxf(m, m2);
  auto shift = [&](float from, float& ss, float& tt) {
    if (from != mm) {
      const float da = (from - mm) * kLog2e, f = fast_exp2(da);
      tt = fmaf(fmaxf(da, kFloor), ss, tt) * f;
      ss *= f;
    }
  };
  shift(m, s, t);
  shift(m2, s2, t2);
  m = mm;
  s += s2;
  t += t2;
}

// a row's results from its sums and its `top` best keys (LDS), by one thread or
// more of a workgroup
template <typename T>
__device__ __forceinline__ void finish_row(const T* x, long row, long target, int V, int top, long ignore,
                                           float m, float s, float t, const uint64_t* best,
                                           float* logprob, float* entropy, float* stats,
                                           int64_t* top_ids, float* top_lp) {
  if (m == -__builtin_huge_valf()) s = __builtin_nanf("");   // no finite logit
  const float l2s = log2f(s);
  // roundings keep on their side of 0 (and NaN stays)
  auto log_p = [&](float v) {
    const float lp = static_cast<float>((static_cast<double>(v) - m) - kLn2 * l2s);
    return lp > 0.0f ? 0.0f : lp;
  };
  if (threadIdx.x == 0) {
    float lp = 0.0f;
    if (target != ignore)
      lp = target >= 0 && target < V ? log_p(to_f32(x[target])) : __builtin_nanf("");
    const float h = static_cast<float>(kLn2) * (l2s - t / s);
    logprob[row] = lp;
    entropy[row] = h < 0.0f ? 0.0f : h;
    if (stats) {
      stats[2 * row] = m;
      stats[2 * row + 1] = l2s;
    }
  }
  if (static_cast<int>(threadIdx.x) < top) {
    const uint64_t key = best[threadIdx.x];
    top_ids[row * top + threadIdx.x] = static_cast<int64_t>(~static_cast<uint32_t>(key));
    top_lp[row * top + threadIdx.x] = log_p(value_of(static_cast<uint32_t>(key >> 32)));
  }
}

// Few long rows: their pieces go to gridDim.y workgroups each (SPLIT), whose sums
// and best keys the join kernel takes from the workspace: (rows, splits) of
// SplitSums, then (rows, splits, top) keys, those behind a split's count not
// written.
struct SplitSums {
  float m, s, t;
  int count;
};

template <typename T, int NT, int P, bool TOP, int WPE, bool SPLIT>
__global__ __launch_bounds__(NT, WPE) void token_logprobs_kernel(
    const T* __restrict__ logits, long ld, const int64_t* __restrict__ targets, int V, int top,
    long ignore, float* __restrict__ logprob, float* __restrict__ entropy,
    float* __restrict__ stats, int64_t* __restrict__ top_ids, float* __restrict__ top_lp,
    SplitSums* __restrict__ split, uint64_t* __restrict__ split_keys) {
  using Raw = typename RawOf<T>::type;
  constexpr int NW = NT / 64, CH = NT * P * 8;   // logits of a piece
  constexpr float kInf = __builtin_huge_valf();
  __shared__ float red[NW];
  __shared__ float2 red2[NW];
  __shared__ float gmax[TOP ? NW : 1][64];
  __shared__ uint64_t list[TOP ? kList + kMaxTop : 1];
  __shared__ uint64_t best[TOP ? kMaxTop : 1];
  __shared__ int wtot[NW];
  __shared__ int hist[TOP ? 256 : 1];
  __shared__ int count;
  __shared__ uint32_t bound;
  const long row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const T* x = logits + row * ld;
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));

  const __amdgpu_buffer_rsrc_t rsrc = row_rsrc(x, off, V);

  float m = -kInf, s = 0.0f, t = 0.0f;
  int nbest = 0;
  (void)nbest;
  const int step = SPLIT ? CH * static_cast<int>(gridDim.y) : CH;
  for (int base = (SPLIT ? static_cast<int>(blockIdx.y) * CH : 0) - off; base < V; base += step) {
    Raw raw[P];
#pragma unroll
    for (int p = 0; p < P; ++p) load8(rsrc, base + (p * NT + tid) * 8, off, raw[p]);
    if (base < 0 || base + CH > V) {   // (uniform) a row's ends
#pragma unroll
      for (int p = 0; p < P; ++p) edge8(base + (p * NT + tid) * 8, V, raw[p]);
    }
    float mx = -kInf, pm[TOP ? P : 1];   // the thread's maximum, and each octet's
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if constexpr (TOP) {
        pm[p] = max8(raw[p], -kInf);
        mx = fmaxf(mx, pm[p]);
      } else {
        mx = max8(raw[p], mx);
      }
    }
#pragma unroll
    for (int p = 0; p < P; ++p) opaque(raw[p]);
    float mc;
    if constexpr (TOP) {
      gmax[wid][lane] = mx;
      __syncthreads();
      float g = gmax[0][lane];
#pragma unroll
      for (int i = 1; i < NW; ++i) g = fmaxf(g, gmax[i][lane]);
      if (wid == 0) {
        // T, the least group maximum with fewer than top larger ones (-inf for a
        // group without logits); the other waves go on
        const uint32_t v = order_of(g);
        int larger = 0;
#pragma unroll
        for (int i = 0; i < 64; ++i) larger += static_cast<uint32_t>(__builtin_amdgcn_readlane(v, i)) > v ? 1 : 0;
        uint32_t least = larger < top ? v : kOrderNan;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1)
          least = min(least, static_cast<uint32_t>(__shfl_xor(static_cast<int>(least), o, 64)));
        if (lane == 0) {
          bound = least;
          count = 0;
        }
      }
      mc = wave_max(g);
    } else {
      mc = block_max<NW>(mx, red);
    }
    // a piece of -inf alone (or with NaN) is taken against 0: its terms are 0 (or NaN)
    const float off_max = mc == -kInf ? 0.0f : mc;
    float sc = 0.0f, tc = 0.0f;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float a = (elem(raw[p], i) - off_max) * kLog2e;
        const float e = fast_exp2(a);
        sc += e;
        tc = fmaf(fmaxf(a, kFloor), e, tc);
      }
#pragma unroll
    for (int p = 0; p < P; ++p) opaque(raw[p]);
    block_sum2<NW>(sc, tc, red2);
    join_sums(m, s, t, mc, sc, tc);

    if constexpr (TOP) {
      if constexpr (NW == 1) __syncthreads();   // bound, count (block_sum2's barrier elsewhere)
      // L: logits whose order is L or above are candidates.  Those of -inf are
      // not, nor those that the pieces before beat (or equal: they came first).
      uint32_t L = max(bound, kOrderLow + 1u), tie = kOrderLow;
      bool ties = bound <= kOrderLow;   // those of -inf may be among the best
      if (nbest == top && static_cast<uint32_t>(best[top - 1] >> 32) >= bound) {
        L = max(L, static_cast<uint32_t>(best[top - 1] >> 32) + 1u);   // (0 behind NaN: see below)
        ties = false;
      }
      auto file = [&](float v, int j) {
        const int at = atomicAdd(&count, 1);
        if (at < kList) list[at] = static_cast<uint64_t>(order_of(v)) << 32 | ~static_cast<uint32_t>(j);
      };
      const bool none = nbest == top && static_cast<uint32_t>(best[top - 1] >> 32) == kOrderNan;
      // a row with NaN (its sums tell) is left to the pass below, as is a list
      // that only NaN could enter
      const bool nan = sc != sc || L > kOrderInf;
      if (!none && !nan) {
        const float lv = value_of(L);
#pragma unroll
        for (int p = 0; p < P; ++p) {
          if (pm[p] >= lv) {   // few octets: about one a candidate
            Raw r = raw[p];
            opaque(r);   // (else pick() makes the array one in memory)
            uint32_t hit = 0u;
#pragma unroll
            for (int i = 0; i < 8; ++i) hit |= elem(r, i) >= lv ? 1u << i : 0u;
            for (; hit; hit &= hit - 1u) {
              const int i = __builtin_ctz(hit);
              file(pick(r, i), base + (p * NT + tid) * 8 + i);
            }
          }
        }
      }
      __syncthreads();
      int nl = count;
      const int j0 = max(base, 0), j1 = min(base + CH, V);
      if (nl > kList || (nan && !none)) {
        // too many: the piece's exact top-th order, digit by digit from the top,
        // the row read again
        uint32_t pre = 0u;
        int need = min(top, j1 - j0);   // of the logits whose digits so far are pre
#pragma unroll 1
        for (int d = 24; d >= 0; d -= 8) {
          __syncthreads();
          if (tid < 64)
            for (int i = tid; i < 256; i += 64) hist[i] = 0;
          __syncthreads();
#pragma unroll 1
          for (int j = j0 + tid; j < j1; j += NT) {
            const uint32_t o = order_of(to_f32(x[j]));
            if (d == 24 || o >> (d + 8) == pre >> (d + 8)) atomicAdd(&hist[o >> d & 255u], 1);
          }
          __syncthreads();
          if (wid == 0) {   // lane: digits 255 - 4 lane .. - 3, from the top
            int h[4], c = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              h[i] = hist[255 - 4 * lane - i];
              c += h[i];
            }
            int above = wave_incl_scan(c, lane) - c;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (above < need && above + h[i] >= need) {
                bound = pre | static_cast<uint32_t>(255 - 4 * lane - i) << d;
                wtot[0] = need - above;
              }
              above += h[i];
            }
          }
          __syncthreads();
          pre = bound;
          need = wtot[0];
        }
        // above it there are fewer than top; those equal to it follow by index
        ties = ties || pre >= L;
        if (pre >= L) tie = pre;
        __syncthreads();
        if (tid == 0) count = 0;
        __syncthreads();
#pragma unroll 1
        for (int j = j0 + tid; j < j1; j += NT) {
          const float v = to_f32(x[j]);
          const uint32_t o = order_of(v);
          if (o > pre && o >= L) file(v, j);
        }
        __syncthreads();
        nl = count;
      }
      if (ties && nl < top) {
        int got = nl;
#pragma unroll 1
        for (int jb = j0; jb < j1 && got < top; jb += NT) {
          const int j = jb + tid;
          const bool eq = j < j1 && order_of(to_f32(x[j])) == tie;
          int total;
          const int at = got + block_scan<NW>(eq ? 1 : 0, wtot, total);
          if (eq && at < top) list[at] = static_cast<uint64_t>(tie) << 32 | ~static_cast<uint32_t>(j);
          got = min(top, got + total);
        }
        nl = got;
        __syncthreads();   // the list is whole
      }
      if (nbest > 0) {
        __syncthreads();
        if (tid < nbest) list[nl + tid] = best[tid];
        nl += nbest;
        __syncthreads();
      }
      // eight threads a candidate count the larger ones
      for (int a = tid >> 3; a < nl; a += NT / 8) {
        const uint64_t key = list[a];
        int rank = 0;
#pragma unroll 2
        for (int b = tid & 7; b < nl; b += 8) rank += list[b] > key ? 1 : 0;
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) rank += __shfl_xor(rank, o, 64);
        if (rank < top && (tid & 7) == 0) best[rank] = key;
      }
      nbest = min(nl, top);
      __syncthreads();
    }
  }
  if constexpr (SPLIT) {
    const long at = row * gridDim.y + blockIdx.y;
    if (tid == 0) split[at] = SplitSums{m, s, t, nbest};
    if constexpr (TOP) {
      if (tid < nbest) split_keys[at * top + tid] = best[tid];
    }
  } else {
    finish_row(x, row, targets[row], V, TOP ? top : 0, ignore, m, s, t, best, logprob, entropy, stats,
               top_ids, top_lp);
  }
}

template <typename T>
__global__ __launch_bounds__(64) void token_logprobs_join_kernel(
    const T* __restrict__ logits, long ld, const int64_t* __restrict__ targets, int V, int top,
    long ignore, float* __restrict__ logprob, float* __restrict__ entropy,
    float* __restrict__ stats, int64_t* __restrict__ top_ids, float* __restrict__ top_lp,
    const SplitSums* __restrict__ split, const uint64_t* __restrict__ split_keys, int splits) {
  __shared__ uint64_t list[2 * kMaxTop], best[kMaxTop];
  const long row = blockIdx.x;
  const int lane = threadIdx.x;
  float m = -__builtin_huge_valf(), s = 0.0f, t = 0.0f;
  int nbest = 0;
  for (int p = 0; p < splits; ++p) {
    const long at = row * splits + p;
    const SplitSums q = split[at];
    join_sums(m, s, t, q.m, q.s, q.t);
    if (top == 0) continue;
    if (lane < nbest) list[lane] = best[lane];
    if (lane < q.count) list[nbest + lane] = split_keys[at * top + lane];
    __syncthreads();
    const int nl = nbest + q.count;
    for (int a = lane; a < nl; a += 64) {
      int rank = 0;
      for (int b = 0; b < nl; ++b) rank += list[b] > list[a] ? 1 : 0;
      if (rank < top) best[rank] = list[a];
    }
    nbest = min(nl, top);
    __syncthreads();
  }
  finish_row(logits + row * ld, row, targets[row], V, top, ignore, m, s, t, best, logprob, entropy, stats,
             top_ids, top_lp);
}

// Gradient.  Workgroup (row, piece of 256 * 8 * kGradP logits); x and dx share
// their offset from a 16-byte boundary (VEC), else single elements.  The stores are
// non-temporal: forward and backward of 8192 x 32000 bf16 take 285 us so and 315
// without, 1500 x 32003 fp32 104 and 124; with the product that reads the gradient
// behind them the two are level (512 to 8192 rows), with a sum 148 and 160.
constexpr int kGradP = 4;
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void token_logprobs_bwd_kernel(
    const T* __restrict__ logits, long ld, const int64_t* __restrict__ targets, int V, int top,
    long ignore, const float* __restrict__ entropy, const float* __restrict__ stats,
    const int64_t* __restrict__ top_ids, const float* __restrict__ g_lp,
    const float* __restrict__ g_h, const float* __restrict__ g_top, T* __restrict__ dx, long ldd) {
  using Raw = typename RawOf<T>::type;
  constexpr int CH = 256 * 8 * kGradP;
  const long row = blockIdx.x;
  const int tid = threadIdx.x;
  const T* x = logits + row * ld;
  T* o = dx + row * ldd;
  const int off = VEC ? static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T)) : 0;
  const int base = static_cast<int>(blockIdx.y) * CH - off;
  const __amdgpu_buffer_rsrc_t rsrc = row_rsrc(x, off, V);
  const float m = stats[2 * row], l2s = stats[2 * row + 1], H = entropy[row];
  const long tg = targets[row];
  const bool asked = tg != ignore;
  float a = asked && g_lp ? g_lp[row] : 0.0f;
  if (asked && g_lp && (tg < 0 || tg >= V)) a = __builtin_nanf("");
  const float h = g_h ? g_h[row] : 0.0f;
  float all = a;
  bool silent = !asked && h == 0.0f;   // zeros, whatever the row holds (a padded place, say)
  if (g_top)
    for (int k = 0; k < top; ++k) {
      all += g_top[row * top + k];
      silent = silent && g_top[row * top + k] == 0.0f;
    }
  const float hl = h * static_cast<float>(kLn2), c = fmaf(h, H, all);   // a + sum b + h (log p + H) = hl log2 p + c
  auto grad = [&](float xv) {
    const float lp = fmaf(xv - m, kLog2e, -l2s);
    return silent ? 0.0f : -fast_exp2(lp) * fmaf(hl, fmaxf(lp, kFloor), c);
  };
#pragma unroll
  for (int q = 0; q < kGradP; ++q) {
    const int j0 = base + (q * 256 + tid) * 8;
    if (j0 >= V) continue;
    if (VEC && j0 >= 0 && j0 + 8 <= V) {
      Raw raw;
      load8(rsrc, j0, off, raw);
      float r[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = grad(elem(raw, i));
      if (static_cast<unsigned long>(tg - j0) < 8ul) {
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] += tg - j0 == i ? a : 0.0f;
      }
      if constexpr (sizeof(T) == 2) {
        typedef uint32_t v4u __attribute__((ext_vector_type(4)));
        __builtin_nontemporal_store(v4u{pack_bf16x2(r[0], r[1]), pack_bf16x2(r[2], r[3]),
                                        pack_bf16x2(r[4], r[5]), pack_bf16x2(r[6], r[7])},
                                    reinterpret_cast<v4u*>(o + j0));
      } else {
        st_nt(reinterpret_cast<float4*>(o + j0), make_float4(r[0], r[1], r[2], r[3]));
        st_nt(reinterpret_cast<float4*>(o + j0 + 4), make_float4(r[4], r[5], r[6], r[7]));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (j0 + i >= 0 && j0 + i < V)
          o[j0 + i] = from_f32<T>(grad(to_f32(x[j0 + i])) + (j0 + i == tg ? a : 0.0f));
    }
  }
  if (g_top) {   // (uniform) the alternatives' own terms, once all is written
    __syncthreads();
    if (tid < top) {
      const long j = top_ids[row * top + tid];
      if (j >= base && j >= 0 && j < V && j < base + CH)
        o[j] = from_f32<T>(grad(to_f32(x[j])) + (j == tg ? a : 0.0f) + g_top[row * top + tid]);
    }
  }
}

constexpr int kLong = 512 * 64;    // logits of the largest piece
constexpr int kFewRows = 512;      // two workgroups a CU
constexpr int kMaxSplits = 16;

// workgroups for each row: rows of several pieces, too few to fill the chip, are
// split: their pieces side by side and a second launch in place of one after
// the other (1 x 131072 bf16, 20 alternatives: 18 us, 22 unsplit; 64 x 50000
// level at 14)
int row_splits(long rows, int V) {
  return rows < kFewRows && V > kLong ? min((V + 7 + kLong - 1) / kLong, kMaxSplits) : 1;
}

template <typename T, bool TOP>
void launch_logprobs(const void* logits, long ld, const int64_t* targets, long rows, int V, int top,
                     long ignore, float* logprob, float* entropy, float* stats, int64_t* top_ids,
                     float* top_lp, void* workspace, hipStream_t s) {
  const int splits = row_splits(rows, V);
  auto* sums = static_cast<SplitSums*>(workspace);
  auto* keys = reinterpret_cast<uint64_t*>(sums + rows * splits);
  auto go = [&](auto kern, int nt) {
    hipLaunchKernelGGL(kern, dim3(rows, splits), dim3(nt), 0, s, static_cast<const T*>(logits), ld,
                       targets, V, top, ignore, logprob, entropy, stats, top_ids, top_lp, sums, keys);
  };
  // waves a SIMD that the registers allow
  constexpr int kW = sizeof(T) == 4 ? 4 : TOP ? 6 : 8;
  if (splits > 1) {
    go(token_logprobs_kernel<T, 512, 8, TOP, 4, true>, 512);
    hipLaunchKernelGGL(token_logprobs_join_kernel<T>, dim3(rows), dim3(64), 0, s,
                       static_cast<const T*>(logits), ld, targets, V, top, ignore, logprob, entropy,
                       stats, top_ids, top_lp, sums, keys, splits);
  } else if (V <= 64 * 64) {
    go(token_logprobs_kernel<T, 64, 8, TOP, kW, false>, 64);
  } else if (V <= 256 * 64 || (TOP && rows >= kFewRows)) {
    // with alternatives the barriers of four waves cost less than those of eight:
    // 8192 x 32000, 20 of them, 120 us in two pieces, 139 in one (91 without any:
    // 86 are the bytes); 4 rows, 8 of them, take 11 us and 9
    go(token_logprobs_kernel<T, 256, 8, TOP, kW, false>, 256);
  } else {
    go(token_logprobs_kernel<T, 512, 8, TOP, 4, false>, 512);
  }
}

int logprobs_check(const char* who, int dtype, const void* logits, long ld, const int64_t* targets,
                   long rows, int V, int top) {
  SA_CHECK_ARG(dtype == kF32 || dtype == kBF16, "%s: dtype %d", who, dtype);
  // (2^32 threads a grid, up to 512 a row)
  SA_CHECK_ARG(rows >= 0 && rows < (1L << 23) && V > 0 && V <= (1 << 28) && ld >= V,
               "%s: bad sizes rows=%ld vocab=%d row stride=%ld", who, rows, V, ld);
  SA_CHECK_ARG(top >= 0 && top <= kMaxTop && top <= V, "%s: top %d must be 0..%d and at most the vocab %d",
               who, top, kMaxTop, V);
  SA_CHECK_ARG(rows == 0 || (logits && targets), "%s: null pointer", who);
  SA_CHECK_ARG((reinterpret_cast<uintptr_t>(logits) & (dtype == kF32 ? 3 : 1)) == 0,
               "%s: logits are not aligned to their type", who);
  return 0;
}

}  // namespace
}  // namespace sa

extern "C" size_t sa_token_logprobs_workspace_size(long rows, int vocab, int top) {
  if (rows <= 0 || vocab <= 0 || top < 0) return 0;
  const size_t splits = sa::row_splits(rows, vocab);
  return splits == 1 ? 0 : rows * splits * (sizeof(sa::SplitSums) + sizeof(uint64_t) * top);
}

extern "C" int sa_token_logprobs_fwd(int dtype, const void* logits, long ld, const int64_t* targets,
                                     long rows, int vocab, int top, long ignore_index,
                                     float* logprob, float* entropy, float* stats,
                                     int64_t* top_ids, float* top_logprobs, void* workspace,
                                     size_t workspace_bytes, void* stream) {
  const char* who = "sa_token_logprobs_fwd";
  if (const int rc = sa::logprobs_check(who, dtype, logits, ld, targets, rows, vocab, top)) return rc;
  if (rows == 0) return 0;
  SA_CHECK_ARG(logprob && entropy && (top == 0 || (top_ids && top_logprobs)), "%s: null pointer",
               who);
  const size_t need = sa_token_logprobs_workspace_size(rows, vocab, top);
  SA_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need), "%s: workspace %zu B < %zu B", who,
               workspace_bytes, need);
  SA_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "%s: workspace is not aligned", who);
  hipStream_t s = static_cast<hipStream_t>(stream);
  sa::ProfScope prof_("token_logprobs", s);
  auto go = [&](auto tc) {
    using T = decltype(tc);
    if (top > 0)
      sa::launch_logprobs<T, true>(logits, ld, targets, rows, vocab, top, ignore_index, logprob,
                                   entropy, stats, top_ids, top_logprobs, workspace, s);
    else
      sa::launch_logprobs<T, false>(logits, ld, targets, rows, vocab, top, ignore_index, logprob,
                                    entropy, stats, top_ids, top_logprobs, workspace, s);
  };
  dtype == sa::kF32 ? go(float{}) : go(sa::bf16{});
  SA_CHECK_LAUNCH("token_logprobs");
  return 0;
}

extern "C" int sa_token_logprobs_bwd(int dtype, const void* logits, long ld, const int64_t* targets,
                                     long rows, int vocab, int top, long ignore_index,
                                     const float* entropy, const float* stats,
                                     const int64_t* top_ids, const float* g_logprob,
                                     const float* g_entropy, const float* g_top, void* dlogits,
                                     long ldd, void* stream) {
  const char* who = "sa_token_logprobs_bwd";
  if (const int rc = sa::logprobs_check(who, dtype, logits, ld, targets, rows, vocab, top)) return rc;
  if (rows == 0) return 0;
  SA_CHECK_ARG(entropy && stats && dlogits && ldd >= vocab && (!g_top || (top > 0 && top_ids)),
               "%s: null pointer or row stride %ld", who, ldd);
  hipStream_t s = static_cast<hipStream_t>(stream);
  sa::ProfScope prof_("token_logprobs_bwd", s);
  const int size = dtype == sa::kF32 ? 4 : 2;
  const uintptr_t px = reinterpret_cast<uintptr_t>(logits), pd = reinterpret_cast<uintptr_t>(dlogits);
  SA_CHECK_ARG(pd % size == 0, "%s: dlogits are not aligned to their type", who);
  // every row of x and dx equally far from a 16-byte boundary
  const bool vec = ((px ^ pd) & 15) == 0 && ((ld - ldd) * size) % 16 == 0;
  constexpr int CH = 256 * 8 * sa::kGradP;
  const int cols = static_cast<int>((vocab + 7L + CH - 1) / CH);   // up to 7 elements of offset
  SA_CHECK_ARG(cols <= 65535, "%s: vocab %d too large", who, vocab);
  auto go = [&](auto kern, auto tc) {
    using T = decltype(tc);
    hipLaunchKernelGGL(kern, dim3(rows, cols), dim3(256), 0, s, static_cast<const T*>(logits), ld,
                       targets, vocab, top, ignore_index, entropy, stats, top_ids, g_logprob,
                       g_entropy, g_top, static_cast<T*>(dlogits), ldd);
  };
  if (dtype == sa::kF32)
    vec ? go(sa::token_logprobs_bwd_kernel<float, true>, float{}) : go(sa::token_logprobs_bwd_kernel<float, false>, float{});
  else
    vec ? go(sa::token_logprobs_bwd_kernel<sa::bf16, true>, sa::bf16{}) : go(sa::token_logprobs_bwd_kernel<sa::bf16, false>, sa::bf16{});
  SA_CHECK_LAUNCH("token_logprobs_bwd");
  return 0;
}
