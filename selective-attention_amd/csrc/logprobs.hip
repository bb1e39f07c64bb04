// Log probabilities of given tokens with the distribution's entropy, its largest
// alternatives, and the gradient (gfx950).  For a row x of V logits, with
// m = max x, d_j = x_j - m, s = sum_j e^d_j, t = sum_j d_j e^d_j:
//
//   log p_j = d_j - log s,   H = -sum_j p_j log p_j = log s - t / s
//   d/dx_j  (a log p_i + h H + sum_k b_k log p_{i_k})
//         = a [j = i] + sum_k b_k [j = i_k] - p_j (a + sum_k b_k + h (log p_j + H))
//
// All in fp32.  Both directions are bound by the bytes of the logits: the
// forward reads them once, the backward reads them and writes the gradient.
//
// Forward: one workgroup a row, which stands in registers (64 logits a thread)
// while its maximum, then the sums, then the alternatives are taken, so that no
// running maximum rescales sums inside a piece; longer rows go in pieces of NT
// * 64 logits, joined by the maximum.
//
// Alternatives, k of them in the order of (value, lowest index first).  Among
// the 64 maxima of 64 disjoint groups of the piece's logits the k-th largest,
// T, is at most the k-th largest logit; logits above T, some 1.2 k on average,
// go to a list in LDS, and ties at T, where the list is shorter than k, in the
// order of their index.  A list that overflows (values sorted against the
// groups) has T replaced by the piece's exact k-th value, by bisection over
// the float's order.  A candidate's place is the number of larger ones.
#include "common.h"
#include "prof.h"

namespace sa {
namespace {

constexpr int kMaxTop = 64;
constexpr int kList = 512;   // candidates of a piece
// e^d is 0 in fp32 from here down: a logit of -inf is taken as this in d e^d,
// which is then 0 and stays so under any factor
constexpr float kFloor = -128.0f;

constexpr uint32_t kOrderNan = 0xffffffffu, kOrderInf = 0xff800000u;
// floats in the order of their values as unsigned numbers above 0: -inf lowest,
// NaN highest, both zeros the same
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return x != x ? kOrderNan : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t o) {
  return o == kOrderNan ? __builtin_nanf("") : __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}

// eight logits j0 .. j0 + 7 of a row of V at x, x + j0 on a 16-byte boundary;
// those outside the row are not read and stand as -inf
struct Raw8f {
  float4 a, b;
};
__device__ __forceinline__ void load8(const bf16* x, long j0, int V, uint4& raw) {
  if (j0 >= 0 && j0 + 8 <= V) {
    raw = *reinterpret_cast<const uint4*>(x + j0);
  } else {
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = j0 + i >= 0 && j0 + i < V ? x[j0 + i].x : 0xff80u;
    raw = uint4{u[0] | u[1] << 16, u[2] | u[3] << 16, u[4] | u[5] << 16, u[6] | u[7] << 16};
  }
}
__device__ __forceinline__ void load8(const float* x, long j0, int V, Raw8f& raw) {
  if (j0 >= 0 && j0 + 8 <= V) {
    raw.a = *reinterpret_cast<const float4*>(x + j0);
    raw.b = *reinterpret_cast<const float4*>(x + j0 + 4);
  } else {
    float u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) u[i] = j0 + i >= 0 && j0 + i < V ? x[j0 + i] : -__builtin_huge_valf();
    raw.a = make_float4(u[0], u[1], u[2], u[3]);
    raw.b = make_float4(u[4], u[5], u[6], u[7]);
  }
}
__device__ __forceinline__ float elem(const uint4& r, int i) {
  const uint32_t w = (i >> 1) == 0 ? r.x : (i >> 1) == 1 ? r.y : (i >> 1) == 2 ? r.z : r.w;
  return (i & 1) ? bf16hi_to_f32(w) : bf16lo_to_f32(w);
}
__device__ __forceinline__ float elem(const Raw8f& r, int i) {
  const float4& q = i < 4 ? r.a : r.b;
  return (i & 3) == 0 ? q.x : (i & 3) == 1 ? q.y : (i & 3) == 2 ? q.z : q.w;
}
template <typename T> struct RawOf;
template <> struct RawOf<bf16> { using type = uint4; };
template <> struct RawOf<float> { using type = Raw8f; };

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
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = wave_sum(v);
  if constexpr (NW > 1) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < NW; ++i) v += red[i];
  }
  return v;
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

template <typename T, int NT, bool TOP>
__global__ __launch_bounds__(NT) void token_logprobs_kernel(
    const T* __restrict__ logits, long ld, const int64_t* __restrict__ targets, int V, int top,
    long ignore, float* __restrict__ logprob, float* __restrict__ entropy,
    float* __restrict__ stats, int64_t* __restrict__ top_ids, float* __restrict__ top_lp) {
  using Raw = typename RawOf<T>::type;
  constexpr int NW = NT / 64, P = 8, CH = NT * P * 8;   // logits of a piece
  __shared__ float red[NW];
  __shared__ float gmax[NW][64];
  __shared__ uint64_t list[TOP ? kList + kMaxTop : 1];
  __shared__ uint64_t best[kMaxTop];
  __shared__ int wtot[NW];
  __shared__ int count;
  __shared__ uint32_t bound;
  const long row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const T* x = logits + row * ld;
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));

  float m = -__builtin_huge_valf(), s = 0.0f, t = 0.0f;
  int nbest = 0;
  for (long base = -off; base < V; base += CH) {
    Raw raw[P];
#pragma unroll
    for (int p = 0; p < P; ++p) load8(x, base + (p * NT + tid) * 8, V, raw[p]);
    float mx = -__builtin_huge_valf();
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = fmaxf(mx, elem(raw[p], i));
    const float mc = block_max<NW>(mx, red);
    // a piece of -inf alone (or with NaN) is taken against 0: its terms are 0 (or NaN)
    const float ref = mc == -__builtin_huge_valf() ? 0.0f : mc;
    float sc = 0.0f, tc = 0.0f;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float d = elem(raw[p], i) - ref;
        const float e = fast_exp2(d * kLog2e);
        sc += e;
        tc += fmaxf(d, kFloor) * e;
      }
    sc = block_sum<NW>(sc, red);
    tc = block_sum<NW>(tc, red);
    // join with the pieces before: against the larger maximum
    const float mn = fmaxf(m, mc);
    auto shift = [&](float from, float& ss, float& tt) {
      if (from != -__builtin_huge_valf() && from != mn) {
        const float dm = from - mn, f = fast_exp2(dm * kLog2e);
        tt = (tt + fmaxf(dm, kFloor) * ss) * f;
        ss *= f;
      }
    };
    shift(m, s, t);
    shift(mc, sc, tc);
    s += sc;
    t += tc;
    m = mn;

    if constexpr (TOP) {
      // T: the top-th largest of the groups' maxima (-inf: a group without
      // logits).  Logits are compared as floats, which takes the two zeros as
      // one; !(x <= T) is true of NaN.
      __syncthreads();
      gmax[wid][lane] = mx;
      __syncthreads();
      if (wid == 0) {
        float g = gmax[0][lane];
#pragma unroll
        for (int i = 1; i < NW; ++i) g = fmaxf(g, gmax[i][lane]);
        const uint32_t v = order_of(g);
        int rank = 0;
#pragma unroll
        for (int i = 0; i < 64; ++i) {
          const uint32_t o = __builtin_amdgcn_readlane(v, i);
          rank += o > v || (o == v && i < lane) ? 1 : 0;
        }
        if (rank == top - 1) bound = v;
        if (lane == 0) count = 0;
      }
      __syncthreads();
      uint32_t T_ = bound;
      bool ties = true;   // logits equal to T may be among the best
      if (nbest == top && static_cast<uint32_t>(best[top - 1] >> 32) >= T_) {
        T_ = static_cast<uint32_t>(best[top - 1] >> 32);
        ties = false;     // equal ones stand behind those of the pieces before
      }
      auto key_of = [&](int p, int i, uint32_t o) {
        const uint32_t j = static_cast<uint32_t>(base + (p * NT + tid) * 8 + i);
        return static_cast<uint64_t>(o) << 32 | ~j;
      };
      auto collect = [&]() {
        if (T_ == kOrderNan) return;   // nothing is above
        const float tv = value_of(T_);
#pragma unroll
        for (int p = 0; p < P; ++p) {
          bool hit = false;
#pragma unroll
          for (int i = 0; i < 8; ++i) hit |= !(elem(raw[p], i) <= tv);
          if (hit) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (!(elem(raw[p], i) <= tv)) {
                const int at = atomicAdd(&count, 1);
                if (at < kList) list[at] = key_of(p, i, order_of(elem(raw[p], i)));
              }
          }
        }
      };
      collect();
      __syncthreads();
      int n = count;
      if (n > kList) {
        // the piece's exact top-th value: the largest T with `top` logits >= T
        uint32_t lo = T_, hi = kOrderNan;
        while (lo < hi) {
          const uint32_t mid = lo + ((hi - lo) >> 1) + 1u;
          const float mv = value_of(mid > kOrderInf ? kOrderInf : mid);
          int c = 0, total;
          if (mid > kOrderInf) {
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
              for (int i = 0; i < 8; ++i) c += elem(raw[p], i) != elem(raw[p], i) ? 1 : 0;
          } else {
#pragma unroll
            for (int p = 0; p < P; ++p)
#pragma unroll
              for (int i = 0; i < 8; ++i) c += !(elem(raw[p], i) < mv) ? 1 : 0;
          }
          block_scan<NW>(c, wtot, total);
          if (total >= top) lo = mid;
          else hi = mid - 1u;
        }
        lo = lo > kOrderInf ? kOrderNan : lo;
        ties = ties || lo > T_;
        T_ = lo;
        if (tid == 0) count = 0;
        __syncthreads();
        collect();
        __syncthreads();
        n = count;   // fewer than top
      }
      if (ties && n < top) {
        // those equal to T, lowest index first (p ascends with the index)
        const float tv = value_of(T_);
        int got = n;
#pragma unroll
        for (int p = 0; p < P; ++p) {
          if (got < top) {   // (uniform)
            uint32_t eq = 0u;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float v = elem(raw[p], i);
              const long j = base + (p * NT + tid) * 8 + i;
              eq |= ((T_ == kOrderNan ? v != v : v == tv) && j >= 0 && j < V) ? 1u << i : 0u;
            }
            int total;
            int at = got + block_scan<NW>(__popc(eq), wtot, total);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (eq >> i & 1u) {
                if (at < top) list[at] = key_of(p, i, T_);
                ++at;
              }
            got = min(top, got + total);
          }
        }
        n = got;
      }
      __syncthreads();
      if (tid < nbest) list[n + tid] = best[tid];
      n += nbest;
      __syncthreads();
      for (int a = tid; a < n; a += NT) {
        const uint64_t key = list[a];
        int rank = 0;
        for (int b = 0; b < n; ++b) rank += list[b] > key ? 1 : 0;
        if (rank < top) best[rank] = key;
      }
      nbest = min(n, top);
      __syncthreads();
    }
  }
  // log p = (x - m) - log s
  const float ls = logf(s);
  if (tid == 0) {
    const long tg = targets[row];
    float lp = 0.0f;
    if (tg != ignore) lp = tg >= 0 && tg < V ? (to_f32(x[tg]) - m) - ls : __builtin_nanf("");
    logprob[row] = lp;
    entropy[row] = ls - t / s;
    stats[2 * row] = m;
    stats[2 * row + 1] = ls;
  }
  if constexpr (TOP) {
    if (tid < top) {
      const uint64_t key = best[tid];
      top_ids[row * top + tid] = static_cast<int64_t>(~static_cast<uint32_t>(key));
      top_lp[row * top + tid] = (value_of(static_cast<uint32_t>(key >> 32)) - m) - ls;
    }
  }
}

// Gradient.  Workgroup (row, piece of 256 * 8 * kGradP logits); x and dx share
// their offset from a 16-byte boundary (VEC), else single elements.
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
  const long base = static_cast<long>(blockIdx.y) * CH - off;
  const float m = stats[2 * row], ls = stats[2 * row + 1], H = entropy[row];
  const long tg = targets[row];
  const bool asked = tg != ignore;
  float a = asked && g_lp ? g_lp[row] : 0.0f;
  if (asked && g_lp && (tg < 0 || tg >= V)) a = __builtin_nanf("");
  const float h = g_h ? g_h[row] : 0.0f;
  float all = a;
  if (g_top)
    for (int k = 0; k < top; ++k) all += g_top[row * top + k];
  auto grad = [&](float xv, long j) {
    const float lp = (xv - m) - ls;
    const float p = fast_exp2(lp * kLog2e);
    const float w = fmaf(h, fmaxf(lp, kFloor) + H, all);
    return (j == tg ? a : 0.0f) - p * w;
  };
#pragma unroll
  for (int q = 0; q < kGradP; ++q) {
    const long j0 = base + (static_cast<long>(q) * 256 + tid) * 8;
    if (j0 >= V) continue;
    if (VEC && j0 >= 0 && j0 + 8 <= V) {
      Raw raw;
      load8(x, j0, V, raw);
      float r[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] = grad(elem(raw, i), j0 + i);
      if constexpr (sizeof(T) == 2) {
        *reinterpret_cast<uint4*>(o + j0) =
            uint4{pack_bf16x2(r[0], r[1]), pack_bf16x2(r[2], r[3]), pack_bf16x2(r[4], r[5]), pack_bf16x2(r[6], r[7])};
      } else {
        *reinterpret_cast<float4*>(o + j0) = make_float4(r[0], r[1], r[2], r[3]);
        *reinterpret_cast<float4*>(o + j0 + 4) = make_float4(r[4], r[5], r[6], r[7]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (j0 + i >= 0 && j0 + i < V) o[j0 + i] = from_f32<T>(grad(to_f32(x[j0 + i]), j0 + i));
    }
  }
  if (g_top) {   // (uniform) the alternatives' own terms, once all is written
    __syncthreads();
    if (tid < top) {
      const long j = top_ids[row * top + tid];
      if (j >= base && j >= 0 && j < V && j < base + CH)
        o[j] = from_f32<T>(grad(to_f32(x[j]), j) + g_top[row * top + tid]);
    }
  }
}

template <typename T, bool TOP>
void launch_logprobs(const void* logits, long ld, const int64_t* targets, long rows, int V, int top,
                     long ignore, float* logprob, float* entropy, float* stats, int64_t* top_ids,
                     float* top_lp, hipStream_t s) {
  auto go = [&](auto kern, int nt) {
    hipLaunchKernelGGL(kern, dim3(rows), dim3(nt), 0, s, static_cast<const T*>(logits), ld, targets, V,
                       top, ignore, logprob, entropy, stats, top_ids, top_lp);
  };
  if (V <= 64 * 64) go(token_logprobs_kernel<T, 64, TOP>, 64);
  else if (V <= 256 * 64) go(token_logprobs_kernel<T, 256, TOP>, 256);
  else go(token_logprobs_kernel<T, 512, TOP>, 512);
}

int logprobs_check(const char* who, int dtype, const void* logits, long ld, const int64_t* targets,
                   long rows, int V, int top) {
  SA_CHECK_ARG(dtype == kF32 || dtype == kBF16, "%s: dtype %d", who, dtype);
  SA_CHECK_ARG(rows >= 0 && rows < (1L << 31) && V > 0 && V <= (1 << 30) && ld >= V,
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

extern "C" int sa_token_logprobs_fwd(int dtype, const void* logits, long ld, const int64_t* targets,
                                     long rows, int vocab, int top, long ignore_index,
                                     float* logprob, float* entropy, float* stats,
                                     int64_t* top_ids, float* top_logprobs, void* stream) {
  const char* who = "sa_token_logprobs_fwd";
  if (const int rc = sa::logprobs_check(who, dtype, logits, ld, targets, rows, vocab, top)) return rc;
  if (rows == 0) return 0;
  SA_CHECK_ARG(logprob && entropy && stats && (top == 0 || (top_ids && top_logprobs)), "%s: null pointer",
               who);
  hipStream_t s = static_cast<hipStream_t>(stream);
  sa::ProfScope prof_("token_logprobs", s);
  auto go = [&](auto tc) {
    using T = decltype(tc);
    if (top > 0)
      sa::launch_logprobs<T, true>(logits, ld, targets, rows, vocab, top, ignore_index, logprob,
                                   entropy, stats, top_ids, top_logprobs, s);
    else
      sa::launch_logprobs<T, false>(logits, ld, targets, rows, vocab, top, ignore_index, logprob,
                                    entropy, stats, top_ids, top_logprobs, s);
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
