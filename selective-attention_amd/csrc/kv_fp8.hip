// Writes of the paged KV cache held in 8 bits (gfx950); its layout is that of
// attention_fp8.hip.
//
// A block (one page of one kv head) is rounded once, when its last token is
// there: with a = max|x| over its values, s = 2^e the smallest power of two with
// a <= 448 s (e >= -126; s = 1 for a = 0), the codes are the e4m3 numbers
// nearest to x / s, ties to even.  A power of two costs no bit of precision
// against a / 448 itself (e4m3 keeps its four significant bits down to 2^-15
// of the top of the range) and makes x / s and code * s exact, so that the one
// rounding is e4m3's, at most 2^-4 of the value.  Tokens whose gate is -inf (a
// key that the head has dropped) are left out of a and stored as 0; the
// block's last token is always in, since it is attended without its gate while
// it is the newest.  Values that are no numbers stay out of a and are stored
// as NaN, infinities with them (e4m3 has none).
//
// Until it is full a row's open block stands in bfloat16 (k_tail, v_tail), in
// the order of a page's elements, so that closing it is elementwise: no token
// is rounded twice, and the codes do not depend on how the tokens came in.
#include "common.h"
#include "prof.h"

#include <algorithm>

namespace sa {
namespace {

// the scale's exponent for the largest finite magnitude with bits `top`
__device__ __forceinline__ int block_exp(uint32_t top) {
  if (top == 0u) return 0;
  // 448 = 1.75 2^8: the mantissa decides between 2^(E - 8) and the next one
  const int e = static_cast<int>(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
  return max(e, -126);
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

using v2u = uint32_t __attribute__((ext_vector_type(2)));

// magnitude bits of a finite bf16, 0 for infinities and NaN
__device__ __forceinline__ uint32_t mag(uint32_t bits16) {
  const uint32_t a = bits16 & 0x7fffu;
  return a < 0x7f80u ? a : 0u;
}
// eight bf16 (in, a uint4) times inv as eight e4m3 codes
__device__ __forceinline__ uint2 encode8(const uint4& x, float inv) {
  const uint32_t u[4] = {x.x, x.y, x.z, x.w};
  uint32_t r[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(bf16lo_to_f32(u[2 * h]) * inv, bf16hi_to_f32(u[2 * h]) * inv, 0, false);
    p = __builtin_amdgcn_cvt_pk_fp8_f32(bf16lo_to_f32(u[2 * h + 1]) * inv, bf16hi_to_f32(u[2 * h + 1]) * inv, p, true);
    r[h] = static_cast<uint32_t>(p);
  }
  return uint2{r[0], r[1]};
}
__device__ __forceinline__ uint32_t mag_max(const uint4& x) {
  const uint32_t u[4] = {x.x, x.y, x.z, x.w};
  uint32_t a = 0u;
#pragma unroll
  for (int i = 0; i < 4; ++i) a = max(a, max(mag(u[i]), mag(u[i] >> 16)));
  return a;
}
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = max(v, static_cast<uint32_t>(__shfl_xor(static_cast<int>(v), o, 64)));
  return v;
}

// One token per row: the token into the open block (and its gate into the page),
// and where that was the block's last slot, the block's codes and scales, a wave
// per (head, keys or values) with its block in registers between the maximum and
// the codes.  Four workgroups a row, since one moves a closing row's 256 KB (8
// heads of 128) through its CU no faster than some 30 GB/s.  The length is read by
// all four and advanced by one, whichever comes last: each sets its bit above
// the length's 27 and so sees the bits set before, and the fourth stores the length
// plus one, without the bits.  None waits for another.
// Bound by latency, one chain of length, page and tail: 64 rows, 8 heads of 128,
// 7 us where no row closes a block, 11 where one does, 13.5 where all do (between
// events; 14.5 and 16.7 with one workgroup a row, and 64 rows of 16 heads, 128
// tokens a block, all closing, 94 against 35).
constexpr int kAppendParts = 4, kLenBits = 27;
template <int D, int PS>
__global__ __launch_bounds__(512) void kv_fp8_append_kernel(
    const bf16* __restrict__ k, const bf16* __restrict__ v, const float* __restrict__ log_gate,
    const int32_t* __restrict__ page_table, int32_t* __restrict__ seq_lens, int heads,
    int max_pages, int num_pages, uint8_t* __restrict__ k_pages, uint8_t* __restrict__ v_pages,
    float* __restrict__ k_scale, float* __restrict__ v_scale, bf16* k_tail, bf16* v_tail,
    float* gate_pages) {
  constexpr int NV = PS * D / 8 / 64;   // 16-byte pieces of a block a lane
  const int row = blockIdx.x / kAppendParts, part = blockIdx.x % kAppendParts, tid = threadIdx.x;
  const int n = heads * D;
  const bf16 *kr = k + static_cast<long>(row) * n, *vr = v + static_cast<long>(row) * n;
  // the loads that wait for no length
  const int e0 = part * 512 + tid;
  const bf16 k0 = e0 < n ? kr[e0] : bf16{}, v0 = e0 < n ? vr[e0] : bf16{};
  __shared__ int len;
  if (tid == 0) {
    const int mine = 1 << (kLenBits + part);
    constexpr int all = ((1 << kAppendParts) - 1) << kLenBits;
    const int old = __hip_atomic_fetch_or(seq_lens + row, mine, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    len = old < 0 ? old : old & ~all;
    if (old >= 0 && ((old | mine) & all) == all)
      __hip_atomic_store(seq_lens + row, len + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  const int t = __builtin_amdgcn_readfirstlane(len);
  if (t < 0) return;
  const int col = min(t / PS, max_pages - 1), s = t % PS;
  const int page = page_table[static_cast<long>(row) * max_pages + col];
  const long tail0 = static_cast<long>(row) * heads * PS * D;
  // an invalid id, or a row past its table: the tail alone is written
  const bool ok = page >= 0 && page < num_pages && t / PS < max_pages;
  const long page0 = static_cast<long>(ok ? page : 0) * heads;
  for (int e = e0; e < n; e += kAppendParts * 512) {
    const int h = e / D, d = e % D;
    const long dst = tail0 + static_cast<long>(h) * PS * D;
    k_tail[dst + s * D + d] = e == e0 ? k0 : kr[e];
    v_tail[dst + d * PS + s] = e == e0 ? v0 : vr[e];
    if (d == 0 && gate_pages && ok)
      gate_pages[(page0 + h) * PS + s] = log_gate[static_cast<long>(row) * heads + h];
  }
  if (s != PS - 1 || !ok) return;
  // The block from the tail, its last token from k and v: the stores above may or
  // may not be there yet, and nothing here depends on them (nor on that token's
  // gate, which does not count).
  const int lane = tid & 63;
  for (int it = part + kAppendParts * __builtin_amdgcn_readfirstlane(tid >> 6); it < 2 * heads; it += kAppendParts * 8) {
    const int h = it >> 1;
    const bool val = it & 1;
    const __amdgpu_buffer_rsrc_t src = make_rsrc((val ? v_tail : k_tail) + tail0 + static_cast<long>(h) * PS * D);
    const __amdgpu_buffer_rsrc_t dst = make_rsrc((val ? v_pages : k_pages) + (page0 + h) * PS * D);
    auto load = [&](int i) __attribute__((always_inline)) {
      return __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(src, 16 * lane, 1024 * i, 0));
    };
    auto store = [&](int i, const uint2& c) __attribute__((always_inline)) {
      __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(v2u, c), dst, 8 * lane, 512 * i, 0);
    };
    const float* gr = gate_pages ? gate_pages + (page0 + h) * PS : nullptr;
    const uint16_t* fresh = reinterpret_cast<const uint16_t*>((val ? vr : kr) + h * D);
    // dropped tokens are 0.  Values: a lane's pieces are all of the same eight
    // tokens (512 % PS = 0), one mask; keys: a piece is of one token.
    uint32_t keep[4] = {~0u, ~0u, ~0u, ~0u};
    if (gr && val) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int tok = (8 * lane) % PS + j;
        if (tok != PS - 1 && gr[tok] == -__builtin_inff()) keep[j >> 1] &= (j & 1) ? 0x0000ffffu : 0xffff0000u;
      }
    }
    const bool last = (8 * lane) % PS == PS - 8;   // values: the piece ends in the last token
    auto piece = [&](uint4 x, int p) __attribute__((always_inline)) {
      if (val) {
        x = uint4{x.x & keep[0], x.y & keep[1], x.z & keep[2], x.w & keep[3]};
        if (last) x.w = (x.w & 0xffffu) | static_cast<uint32_t>(fresh[8 * p / PS]) << 16;
        return x;
      }
      const int tok = 8 * p / D;
      if (tok == PS - 1) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          w[j] = fresh[8 * p % D + 2 * j] | static_cast<uint32_t>(fresh[8 * p % D + 2 * j + 1]) << 16;
        return uint4{w[0], w[1], w[2], w[3]};
      }
      return gr && gr[tok] == -__builtin_inff() ? uint4{0u, 0u, 0u, 0u} : x;
    };
    uint4 x[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i] = load(i);
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      x[i] = piece(x[i], lane + 64 * i);
      top = max(top, mag_max(x[i]));
    }
    const int e = block_exp(wave_umax(top) << 16);
    const float inv = pow2f(-e);
#pragma unroll
    for (int i = 0; i < NV; ++i) store(i, encode8(x[i], inv));
    if (lane == 0) (val ? v_scale : k_scale)[page0 + h] = pow2f(e);
  }
}

// A prompt's tokens.  Block (page slot j of row r, head h): a full page is
// rounded, an open one goes to the row's tail, zeros behind its tokens; the
// page's gates, -inf behind the tokens.  V turns over in LDS.
template <int D, int PS>
__global__ __launch_bounds__(256) void kv_fp8_build_kernel(
    const bf16* __restrict__ k, const bf16* __restrict__ v, long sb, long st, long sh,
    const float* __restrict__ lg, long gb, long gh, long gt, const int32_t* __restrict__ page_table,
    const int32_t* __restrict__ seq_lens, int seqlen, int H, int max_pages, int cols, int num_pages,
    uint8_t* __restrict__ k_pages, uint8_t* __restrict__ v_pages, float* __restrict__ k_scale,
    float* __restrict__ v_scale, bf16* __restrict__ k_tail, bf16* __restrict__ v_tail,
    float* __restrict__ gate_pages) {
  constexpr int NV = PS * D / 8 / 256;   // 16-byte pieces of a block a thread
  constexpr int LDV = D + 8;
  __shared__ __align__(16) bf16 tile[PS * LDV];
  __shared__ uint32_t tops[2][4];
  __shared__ uint8_t drop[PS];
  const int r = blockIdx.x / cols, j = blockIdx.x % cols, h = blockIdx.y;
  const int n = min(max(seq_lens[r], 0), seqlen), t0 = j * PS;
  if (t0 >= n) return;   // (uniform) no token of the row in this page slot
  const int page = page_table[static_cast<long>(r) * max_pages + j];
  if (page < 0 || page >= num_pages) return;
  const int m = min(PS, n - t0);
  const long blk = static_cast<long>(page) * H + h;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  if (tid < PS) {
    bool dead = tid >= m;
    if (gate_pages) {
      const float gv = dead ? -__builtin_inff() : lg[r * gb + h * gh + (t0 + tid) * gt];
      gate_pages[blk * PS + tid] = gv;
      dead = dead || (m == PS && tid != PS - 1 && gv == -__builtin_inff());
    }
    drop[tid] = dead;
  }
  const bf16* kr = k + r * sb + h * sh + t0 * st;
  const bf16* vr = v + r * sb + h * sh + t0 * st;
  uint4 kx[NV], vx[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = tid + 256 * i, tok = e / (D / 8), c8 = e % (D / 8);
    kx[i] = ld16(kr + tok * st + 8 * c8, tok < m);
    vx[i] = ld16(vr + tok * st + 8 * c8, tok < m);
  }
  __syncthreads();   // drop
  uint32_t kt = 0u, vt = 0u;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = tid + 256 * i, tok = e / (D / 8), c8 = e % (D / 8);
    if (drop[tok]) kx[i] = vx[i] = uint4{0u, 0u, 0u, 0u};
    kt = max(kt, mag_max(kx[i]));
    vt = max(vt, mag_max(vx[i]));
    *reinterpret_cast<uint4*>(tile + tok * LDV + 8 * c8) = vx[i];
  }
  kt = wave_umax(kt);
  vt = wave_umax(vt);
  if (lane == 0) {
    tops[0][wid] = kt;
    tops[1][wid] = vt;
  }
  __syncthreads();   // tile, tops
  const bool full = m == PS;
  const int ek = block_exp(max(max(tops[0][0], tops[0][1]), max(tops[0][2], tops[0][3])) << 16);
  const int ev = block_exp(max(max(tops[1][0], tops[1][1]), max(tops[1][2], tops[1][3])) << 16);
  const long tail = (static_cast<long>(r) * H + h) * PS * D;
  if (full && tid == 0) {
    k_scale[blk] = pow2f(ek);
    v_scale[blk] = pow2f(ev);
  }
  const float ki = pow2f(-ek), vi = pow2f(-ev);
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int e = tid + 256 * i;
    if (full)
      reinterpret_cast<uint2*>(k_pages + blk * PS * D)[e] = encode8(kx[i], ki);
    else
      reinterpret_cast<uint4*>(k_tail + tail)[e] = kx[i];
    // eight tokens of one dim of V
    const int d = e / (PS / 8), s8 = e % (PS / 8);
    uint32_t w[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const uint32_t lo = tile[(8 * s8 + 2 * q) * LDV + d].x, hi = tile[(8 * s8 + 2 * q + 1) * LDV + d].x;
      w[q] = lo | (hi << 16);
    }
    const uint4 x = {w[0], w[1], w[2], w[3]};
    if (full)
      reinterpret_cast<uint2*>(v_pages + blk * PS * D)[e] = encode8(x, vi);
    else
      reinterpret_cast<uint4*>(v_tail + tail)[e] = x;
  }
}

int cache_check(const char* who, const void* k, const void* v, const float* log_gate,
                const int32_t* page_table, const int32_t* seq_lens, int batch, int heads,
                int head_dim, int page_size, int max_pages, int num_pages, const void* k_pages,
                const void* v_pages, const float* k_scale, const float* v_scale,
                const void* k_tail, const void* v_tail, const float* gate_pages) {
  SA_CHECK_ARG(batch >= 0 && heads > 0 && heads <= 65535 && max_pages > 0 && num_pages > 0,
               "%s: bad sizes batch=%d heads=%d max_pages=%d num_pages=%d", who, batch, heads,
               max_pages, num_pages);
  SA_CHECK_ARG(head_dim == 64 || head_dim == 128, "%s: head_dim %d not in {64,128}", who, head_dim);
  SA_CHECK_ARG(page_size == 64 || page_size == 128, "%s: page_size %d not in {64, 128}", who,
               page_size);
  SA_CHECK_ARG(static_cast<long>(max_pages) * page_size <= (1L << 30), "%s: max_pages %d too large",
               who, max_pages);
  SA_CHECK_ARG(k && v && page_table && seq_lens && k_pages && v_pages && k_scale && v_scale &&
                   k_tail && v_tail,
               "%s: null pointer", who);
  SA_CHECK_ARG((log_gate != nullptr) == (gate_pages != nullptr),
               "%s: log_gate and gate_pages go together", who);
  SA_CHECK_ARG(((reinterpret_cast<uintptr_t>(k_pages) | reinterpret_cast<uintptr_t>(v_pages) |
                 reinterpret_cast<uintptr_t>(k_tail) | reinterpret_cast<uintptr_t>(v_tail)) & 15) == 0,
               "%s: the pages and the tails must be 16-byte aligned", who);
  return 0;
}

}  // namespace
}  // namespace sa

extern "C" int sa_paged_kv_append_fp8(const void* k, const void* v, const float* log_gate,
                                      const int32_t* page_table, int32_t* seq_lens, int batch,
                                      int heads, int head_dim, int page_size, int max_pages,
                                      int num_pages, void* k_pages, void* v_pages, float* k_scale,
                                      float* v_scale, void* k_tail, void* v_tail,
                                      float* gate_pages, void* stream) {
  if (const int rc = sa::cache_check("sa_paged_kv_append_fp8", k, v, log_gate, page_table, seq_lens,
                                     batch, heads, head_dim, page_size, max_pages, num_pages,
                                     k_pages, v_pages, k_scale, v_scale, k_tail, v_tail, gate_pages))
    return rc;
  SA_CHECK_ARG(static_cast<long>(max_pages) * page_size < (1L << sa::kLenBits) && batch < (1 << 21),
               "sa_paged_kv_append_fp8: table of %d pages x %d rows too large", max_pages, batch);
  if (batch == 0) return 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  sa::ProfScope prof_("kv_fp8_append", s);
  auto launch = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3(batch * sa::kAppendParts), dim3(512), 0, s, static_cast<const sa::bf16*>(k),
                       static_cast<const sa::bf16*>(v), log_gate, page_table, seq_lens, heads,
                       max_pages, num_pages, static_cast<uint8_t*>(k_pages),
                       static_cast<uint8_t*>(v_pages), k_scale, v_scale,
                       static_cast<sa::bf16*>(k_tail), static_cast<sa::bf16*>(v_tail), gate_pages);
  };
  if (head_dim == 64)
    page_size == 64 ? launch(sa::kv_fp8_append_kernel<64, 64>) : launch(sa::kv_fp8_append_kernel<64, 128>);
  else
    page_size == 64 ? launch(sa::kv_fp8_append_kernel<128, 64>) : launch(sa::kv_fp8_append_kernel<128, 128>);
  SA_CHECK_LAUNCH("kv_fp8_append");
  return 0;
}

extern "C" int sa_paged_kv_build_fp8(const void* k, const void* v, long sb, long st, long sh,
                                     const float* log_gate, long gb, long gh, long gt,
                                     const int32_t* page_table, const int32_t* seq_lens, int batch,
                                     int seqlen, int heads, int head_dim, int page_size,
                                     int max_pages, int num_pages, void* k_pages, void* v_pages,
                                     float* k_scale, float* v_scale, void* k_tail, void* v_tail,
                                     float* gate_pages, void* stream) {
  const char* who = "sa_paged_kv_build_fp8";
  if (const int rc = sa::cache_check(who, k, v, log_gate, page_table, seq_lens, batch, heads,
                                     head_dim, page_size, max_pages, num_pages, k_pages, v_pages,
                                     k_scale, v_scale, k_tail, v_tail, gate_pages))
    return rc;
  SA_CHECK_ARG(seqlen >= 0, "%s: seqlen %d", who, seqlen);
  SA_CHECK_ARG(((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) == 0 &&
                   sb % 8 == 0 && st % 8 == 0 && sh % 8 == 0,
               "%s: k / v and their strides must keep 16-byte alignment", who);
  // page slots that can hold tokens
  const int cols = static_cast<int>(std::min<long>(max_pages, (static_cast<long>(seqlen) + page_size - 1) / page_size));
  SA_CHECK_ARG(static_cast<long>(batch) * cols < (1L << 24), "%s: too many pages", who);   // (2^32 threads a grid)
  if (batch == 0 || cols == 0) return 0;
  hipStream_t s = static_cast<hipStream_t>(stream);
  sa::ProfScope prof_("kv_fp8_build", s);
  auto launch = [&](auto kern) {
    hipLaunchKernelGGL(kern, dim3(batch * cols, heads), dim3(256), 0, s,
                       static_cast<const sa::bf16*>(k), static_cast<const sa::bf16*>(v), sb, st, sh,
                       log_gate, gb, gh, gt, page_table, seq_lens, seqlen, heads, max_pages, cols,
                       num_pages, static_cast<uint8_t*>(k_pages), static_cast<uint8_t*>(v_pages),
                       k_scale, v_scale, static_cast<sa::bf16*>(k_tail),
                       static_cast<sa::bf16*>(v_tail), gate_pages);
  };
  if (head_dim == 64)
    page_size == 64 ? launch(sa::kv_fp8_build_kernel<64, 64>) : launch(sa::kv_fp8_build_kernel<64, 128>);
  else
    page_size == 64 ? launch(sa::kv_fp8_build_kernel<128, 64>) : launch(sa::kv_fp8_build_kernel<128, 128>);
  SA_CHECK_LAUNCH("kv_fp8_build");
  return 0;
}
