// Linear layers with 4-bit weights and group scales, for few rows (gfx950).
//
//   y[m, n] = sum_k x[m, k] W[n, k] + bias[n],  W[n, k] = s[n, k / G] (c[n, k] - z[n, k / G])
//
// c in 0..15, G in {32, 64, 128}, z = 8 where no zero points are given.  At
// decode sizes the layer is bound by the bytes of the weights, a quarter of
// bf16's, so the widening must cost less than their loads: a code becomes the
// bf16 number 1 + c / 16 by placing its four bits under the exponent of 1 (one
// shift and one and-or for two codes), exactly, and the group's factors are
// applied to sums in fp32:
//
//   sum_k x (c - z) = 16 (sum_k x (1 + c / 16) - (1 + z / 16) sum_k x)
//
// both sums on the matrix cores (16x16x32, the weights as the A operand, x as
// B; sum_k x as the product with ones, once for all tiles of a wave).  Both are
// rounded on their own, so a result is off by at most (K / 32 + 36) 2^-24 times 16
// (1.94 + 1.94) sum_k s |x_k| before its one rounding to bf16: a share of s |x|,
// not of |x w|, which codes at the zero point do not make smaller.  A group without
// a weight has s = 0 and adds exactly nothing.
//
// Packed weights: tiles of 16 rows and 128 columns, (N / 16, K / 128, 64, 16)
// bytes, so that one 16-byte load a lane is a tile.  Lane 16 g + c holds row c;
// its byte 4 j + i has, in its low and high half, columns 32 j + 8 g + 2 i and
// + 1.  Scales and zero points: (N / 16, groups, 16) bf16, groups = (K / 128)
// 128 / G.  N and K are padded to whole tiles; columns at or behind K meet
// x = 0 and rows behind N are not stored.
#include "common.h"
#include "prof.h"

#include <algorithm>
#include <type_traits>

namespace sa {
namespace {

constexpr int kInt4Segs = 4;
struct Int4Segs {
  const uint4* W[kInt4Segs];
  const bf16* scale[kInt4Segs];
  const bf16* zero[kInt4Segs];
  const bf16* bias[kInt4Segs];
  bf16* y[kInt4Segs];
  int N[kInt4Segs];
  int blk0[kInt4Segs + 1];
  int nseg;
};

// codes of one k-step (8 of a lane, one word) as 1 + c / 16; the operand's
// pairs are codes (q, q + 4), four bits apart by 16 in the word
__device__ __forceinline__ v8bf widen_codes(uint32_t w) {
  constexpr uint32_t kMask = 0x00780078u, kOne = 0x3f803f80u;
  const uint4 r = {((w << 3) & kMask) | kOne, ((w >> 1) & kMask) | kOne, ((w >> 5) & kMask) | kOne,
                   ((w >> 9) & kMask) | kOne};
  return __builtin_bit_cast(v8bf, r);
}
// eight consecutive x in that order: (0, 4), (1, 5), (2, 6), (3, 7)
__device__ __forceinline__ v8bf pair_x(const uint4& x) {
  const uint4 r = {__builtin_amdgcn_perm(x.z, x.x, 0x05040100u), __builtin_amdgcn_perm(x.z, x.x, 0x07060302u),
                   __builtin_amdgcn_perm(x.w, x.y, 0x05040100u), __builtin_amdgcn_perm(x.w, x.y, 0x07060302u)};
  return __builtin_bit_cast(v8bf, r);
}
__device__ __forceinline__ uint32_t mul_pair(uint32_t a, uint32_t b) {
  return pack_bf16x2(bf16lo_to_f32(a) * bf16lo_to_f32(b), bf16hi_to_f32(a) * bf16hi_to_f32(b));
}

// whether the pieces of eight columns stand on 16-byte boundaries and none passes K
__device__ __forceinline__ bool whole_pieces(const bf16* x, int K, int ldx) {
  return ((K | ldx) & 7) == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
}
// J blocks of 128 columns and 16 rows of x, those outside x as 0 (buffer loads,
// whose range check answers for them without a branch), times xscale, rounded to
// bf16, where that is given.  They are read along the rows (16 lanes a row, 4 rows
// a load) and turned into operand order in the wave's own LDS (16 rows of 272
// bytes): loads in operand order take 64 bytes from each of 16 rows, which at K =
// 4096 lie in one channel of the L2 (64 rows, 4096 -> 4096: 13.8 us, turned 10.0;
// 32 rows, 4096 -> 32000: 25.0 and 21.3).
constexpr int kTurnRow = 17;   // uint4
template <int J>
__device__ __forceinline__ void read_rows(uint4 (&v)[J][4], const bf16* x, int row0, int k0, int M, int K, int ldx) {
  const int lane = threadIdx.x & 63;
  if (whole_pieces(x, K, ldx)) {   // (uniform)
    const int bytes = M * ldx * 2;
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<bf16*>(x), static_cast<short>(0), bytes, 0x00020000);
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = row0 + 4 * i + (lane >> 4), k = k0 + 128 * j + 8 * (lane & 15);
        const int at = row < M && k < K ? (row * ldx + k) * 2 : bytes;
        v[j][i] = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0));
      }
    return;
  }
  // from the words that hold them: five, moved by half a word where a row starts in
  // the middle of one, columns at and behind K as 0 (4 rows of 1023, 4383 outputs:
  // 4.0 us, 3.6 of 1024; 32 of 4091, 32000 outputs: 25 and 21; a padded copy in
  // front takes 10 us)
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(x) & 2);
  const int bytes = (off + ((M - 1) * ldx + K) * 2 + 3) & ~3;
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<char*>(reinterpret_cast<const char*>(x) - off), static_cast<short>(0), bytes, 0x00020000);
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = row0 + 4 * i + (lane >> 4), k = k0 + 128 * j + 8 * (lane & 15);
      const int at = row < M && k < K ? off + (row * ldx + k) * 2 : bytes;
      const uint4 a = __builtin_bit_cast(uint4, __builtin_amdgcn_raw_buffer_load_b128(r, at & ~3, 0, 0));
      const uint32_t e = __builtin_amdgcn_raw_buffer_load_b32(r, (at & ~3) + 16, 0, 0);
      const int sh = 8 * (at & 2), n = K - k;
      uint32_t w[4] = {__builtin_amdgcn_alignbit(a.y, a.x, sh), __builtin_amdgcn_alignbit(a.z, a.y, sh),
                       __builtin_amdgcn_alignbit(a.w, a.z, sh), __builtin_amdgcn_alignbit(e, a.w, sh)};
#pragma unroll
      for (int q = 0; q < 4; ++q) w[q] &= n > 2 * q + 1 ? ~0u : n > 2 * q ? 0xffffu : 0u;
      v[j][i] = uint4{w[0], w[1], w[2], w[3]};
    }
}
template <int J>
__device__ __forceinline__ void load_x_rows(uint4 (&v)[J][4], const bf16* x, const bf16* xscale, int row0,
                                            int k0, int M, int K, int ldx) {
  read_rows(v, x, row0, k0, M, K, ldx);
  if (xscale) {
    uint4 f[J][4];
    read_rows(f, xscale, row0, k0, M, K, ldx);
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint4& u = v[j][i];
        u = uint4{mul_pair(u.x, f[j][i].x), mul_pair(u.y, f[j][i].y), mul_pair(u.z, f[j][i].z), mul_pair(u.w, f[j][i].w)};
      }
  }
}
__device__ __forceinline__ void turn_x(v8bf (&xf)[4], const uint4 (&v)[4], uint4* lds) {
  const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) lds[(4 * i + g) * kTurnRow + c] = v[i];
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int j = 0; j < 4; ++j) xf[j] = pair_x(lds[c * kTurnRow + 4 * j + g]);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// A workgroup of NW waves computes R tiles of 16 columns of y for up to 16 CT
// rows of x; the waves take the 128-column blocks of K in turn and their sums
// meet in LDS.
template <int CT, int G, bool Z, int R, int NW>
__global__ __launch_bounds__(64 * NW) void int4_linear_kernel(const bf16* __restrict__ x,
                                                              const bf16* __restrict__ xscale,
                                                              const Int4Segs sg, int M, int K,
                                                              int ldx) {
  constexpr int GN = 128 / G, GS = G / 32;   // groups of a block, k-steps of a group
  constexpr int kPart = NW * R * CT * 64, kTurn = 16 * kTurnRow;   // uint4, a wave's uint4
  __shared__ uint4 smem[NW * kTurn > kPart ? NW * kTurn : kPart];     // x turned, then the sums
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, c = lane & 15, g = lane >> 4;
  const int bid = blockIdx.x;
  int seg = 0;
#pragma unroll
  for (int i = 1; i < kInt4Segs; ++i) seg += (i < sg.nseg && bid >= sg.blk0[i]) ? 1 : 0;
  const int N = sg.N[seg], tiles = (N + 15) >> 4, kb_n = (K + 127) >> 7;
  const int t0 = (bid - sg.blk0[seg]) * R;
  const uint4* W = sg.W[seg];
  const uint2* S = reinterpret_cast<const uint2*>(sg.scale[seg]);
  const uint2* ZP = reinterpret_cast<const uint2*>(sg.zero[seg]);

  v4f acc[R][CT];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < CT; ++t) acc[r][t] = v4f{0.f, 0.f, 0.f, 0.f};
  v8bf ones;
  {
    const uint4 o = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
    ones = __builtin_bit_cast(v8bf, o);
  }
  auto tile_of = [&](int r) { return static_cast<long>(min(t0 + r, tiles - 1)); };   // (behind the last: not stored)

  for (int kb = wid; kb < kb_n; kb += NW) {
    uint4 w[R];
#pragma unroll
    for (int r = 0; r < R; ++r) w[r] = W[(tile_of(r) * kb_n + kb) * 64 + lane];
    uint2 s[R][GN], z[R][GN];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int i = 0; i < GN; ++i) {
        const long at = ((tile_of(r) * kb_n + kb) * GN + i) * 4 + g;
        s[r][i] = S[at];
        if constexpr (Z) z[r][i] = ZP[at];
      }
    v8bf xf[CT][4];
    uint4 xr[CT][1][4];
#pragma unroll
    for (int t = 0; t < CT; ++t) load_x_rows(xr[t], x, xscale, 16 * t, 128 * kb, M, K, ldx);
#pragma unroll
    for (int t = 0; t < CT; ++t) turn_x(xf[t], xr[t][0], smem + wid * kTurn);
#pragma unroll
    for (int i = 0; i < GN; ++i) {
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        v4f xs = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < GS; ++j) xs = mfma_bf16(ones, xf[t][GS * i + j], xs);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const uint32_t wj[4] = {w[r].x, w[r].y, w[r].z, w[r].w};
          v4f d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < GS; ++j) d = mfma_bf16(widen_codes(wj[GS * i + j]), xf[t][GS * i + j], d);
          const float sv[4] = {bf16lo_to_f32(s[r][i].x), bf16hi_to_f32(s[r][i].x), bf16lo_to_f32(s[r][i].y),
                               bf16hi_to_f32(s[r][i].y)};
          float zv[4] = {8.f, 8.f, 8.f, 8.f};
          if constexpr (Z) {
            zv[0] = bf16lo_to_f32(z[r][i].x);
            zv[1] = bf16hi_to_f32(z[r][i].x);
            zv[2] = bf16lo_to_f32(z[r][i].y);
            zv[3] = bf16hi_to_f32(z[r][i].y);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[r][t][e] = fmaf(16.0f * sv[e], fmaf(-(1.0f + 0.0625f * zv[e]), xs[e], d[e]), acc[r][t][e]);
        }
      }
    }
  }
  // lane (c, g) holds columns 4 g + e of the tile for row 16 t + c of x
  float* part = reinterpret_cast<float*>(smem);
  __syncthreads();   // the turned rows are read
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < CT; ++t)
      *reinterpret_cast<float4*>(part + ((wid * R + r) * CT + t) * 256 + c * 16 + 4 * g) =
          make_float4(acc[r][t][0], acc[r][t][1], acc[r][t][2], acc[r][t][3]);
  __syncthreads();
  const bf16* bias = sg.bias[seg];
  bf16* y = sg.y[seg];
  for (int e = tid; e < R * CT * 256; e += 64 * NW) {
    const int row = (e >> 4) % (16 * CT), n = 16 * (t0 + e / (CT * 256)) + (e & 15);
    const float* p = part + e;
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < NW; ++i) v += p[i * R * CT * 256];
    if (row < M && n < N) y[static_cast<long>(row) * N + n] = from_f32<bf16>(v + (bias ? to_f32(bias[n]) : 0.0f));
  }
}

// The same for K up to 8 KW blocks of 128 columns: wave w of a workgroup keeps x
// of its KW blocks in registers, in operand order and with the groups' sums, and
// the workgroup goes through the tiles t, t + gridDim.x, ..., so that only the
// weights are streamed: x is read and put in order once a workgroup, not once a
// tile (4096 -> 32000, group 128, 8 rows: 17.3 us by tiles, 15.8 here; 32 rows: 31.3
// and 21.3; the weights' bytes at 6 TB/s are 11.4 us).  The next tile's codes and factors are
// in flight while this one's are multiplied (two in flight: no faster); the eight
// waves' sums meet in one of two LDS buffers, one barrier a tile.
template <int CT, int G, bool Z, int KW>
__global__ __launch_bounds__(512, CT == 1 && KW < 4 ? 3 : 2) void int4_stream_kernel(
    const bf16* __restrict__ x, const bf16* __restrict__ xscale, const Int4Segs sg, int M, int K,
    int ldx) {
  constexpr int GN = 128 / G, GS = G / 32, NW = 8;
  constexpr int kPart = NW * CT * 256, kTurn = 16 * kTurnRow;   // floats, uint4 a wave
  __shared__ uint4 smem[(NW * kTurn > 2 * kPart / 4) ? NW * kTurn : 2 * kPart / 4];   // x turned, then the sums
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, c = lane & 15, g = lane >> 4;
  const int kb_n = (K + 127) >> 7, kb0 = wid * KW, m0 = blockIdx.y * 16 * CT;
  const int total = sg.blk0[kInt4Segs];   // tiles of all matrices

  struct Tile {
    uint4 w[KW];
    uint2 s[KW * GN], z[Z ? KW * GN : 1];
  };
  auto seg_of = [&](int t) {
    int seg = 0;
#pragma unroll
    for (int i = 1; i < kInt4Segs; ++i) seg += (i < sg.nseg && t >= sg.blk0[i]) ? 1 : 0;
    return seg;
  };
  auto load = [&](int t, Tile& q) __attribute__((always_inline)) {
    const int seg = seg_of(t);
    const long first = static_cast<long>(t - sg.blk0[seg]) * kb_n;
    const uint4* W = sg.W[seg];
    const uint2* S = reinterpret_cast<const uint2*>(sg.scale[seg]);
    const uint2* ZP = reinterpret_cast<const uint2*>(sg.zero[seg]);
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      const long kb = first + min(kb0 + k, kb_n - 1);   // (blocks behind the last meet x = 0)
      q.w[k] = W[kb * 64 + lane];
#pragma unroll
      for (int i = 0; i < GN; ++i) {
        q.s[k * GN + i] = S[(kb * GN + i) * 4 + g];
        if constexpr (Z) q.z[k * GN + i] = ZP[(kb * GN + i) * 4 + g];
      }
    }
  };
  int t = blockIdx.x;   // (gridDim.x <= total)
  const int step = gridDim.x;
  Tile q0, q1;      // one is multiplied, the next in flight
  load(t, q0);

  v8bf xf[CT][KW][4];
  float xs[CT][KW * GN];
  {
    const uint4 o = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
    const v8bf ones = __builtin_bit_cast(v8bf, o);
    uint4 xr[CT][KW][4];
#pragma unroll
    for (int t = 0; t < CT; ++t) load_x_rows(xr[t], x, xscale, m0 + 16 * t, 128 * kb0, M, K, ldx);
#pragma unroll
    for (int t = 0; t < CT; ++t)
#pragma unroll
      for (int k = 0; k < KW; ++k) turn_x(xf[t][k], xr[t][k], smem + wid * kTurn);
#pragma unroll
    for (int t = 0; t < CT; ++t)
#pragma unroll
      for (int i = 0; i < KW * GN; ++i) {
        v4f s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < GS; ++j) s = mfma_bf16(ones, xf[t][i / GN][GS * (i % GN) + j], s);
        xs[t][i] = s[0];   // every row of the product is the same
      }
  }

  __syncthreads();   // the turned rows are read
  int flip = 0;
  auto tile = [&](const Tile& cur, Tile& free) __attribute__((always_inline)) {
    load(min(t + step, total - 1), free);
    v4f acc[CT];
#pragma unroll
    for (int u = 0; u < CT; ++u) acc[u] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < KW; ++k) {
      const uint32_t wj[4] = {cur.w[k].x, cur.w[k].y, cur.w[k].z, cur.w[k].w};
#pragma unroll
      for (int i = 0; i < GN; ++i) {
        const int gi = k * GN + i;
        v4f d[CT];
#pragma unroll
        for (int u = 0; u < CT; ++u) d[u] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < GS; ++j) {
          const v8bf a = widen_codes(wj[GS * i + j]);
#pragma unroll
          for (int u = 0; u < CT; ++u) d[u] = mfma_bf16(a, xf[u][k][GS * i + j], d[u]);
        }
        const float sv[4] = {bf16lo_to_f32(cur.s[gi].x), bf16hi_to_f32(cur.s[gi].x),
                             bf16lo_to_f32(cur.s[gi].y), bf16hi_to_f32(cur.s[gi].y)};
        float zv[4] = {8.f, 8.f, 8.f, 8.f};
        if constexpr (Z) {
          zv[0] = bf16lo_to_f32(cur.z[gi].x);
          zv[1] = bf16hi_to_f32(cur.z[gi].x);
          zv[2] = bf16lo_to_f32(cur.z[gi].y);
          zv[3] = bf16hi_to_f32(cur.z[gi].y);
        }
#pragma unroll
        for (int u = 0; u < CT; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[u][e] = fmaf(16.0f * sv[e], fmaf(-(1.0f + 0.0625f * zv[e]), xs[u][gi], d[u][e]), acc[u][e]);
      }
    }
    float* buf = reinterpret_cast<float*>(smem) + flip * kPart;
#pragma unroll
    for (int u = 0; u < CT; ++u)
      *reinterpret_cast<float4*>(buf + (wid * CT + u) * 256 + c * 16 + 4 * g) = make_float4(acc[u][0], acc[u][1], acc[u][2], acc[u][3]);
    __syncthreads();
    const int seg = seg_of(t), N = sg.N[seg];
    const bf16* bias = sg.bias[seg];
    bf16* y = sg.y[seg];
    for (int e = tid; e < CT * 256; e += 64 * NW) {
      const int row = m0 + (e >> 4), n = 16 * (t - sg.blk0[seg]) + (e & 15);
      float v = 0.0f;
#pragma unroll
      for (int i = 0; i < NW; ++i) v += buf[i * CT * 256 + e];
      if (row < M && n < N) y[static_cast<long>(row) * N + n] = from_f32<bf16>(v + (bias ? to_f32(bias[n]) : 0.0f));
    }
    flip ^= 1;
    t += step;
  };
  // (two copies of the body, so that no register of a load in flight is moved)
  while (true) {
    tile(q0, q1);
    if (t >= total) break;
    tile(q1, q0);
    if (t >= total) break;
  }
}

// the weights in bf16, (N, K) row-major: for many rows, where a plain matrix
// product follows.  One workgroup a tile and 128 columns.
__global__ __launch_bounds__(256) void int4_dequant_kernel(const uint32_t* __restrict__ W,
                                                           const bf16* __restrict__ scale,
                                                           const bf16* __restrict__ zero,
                                                           bf16* __restrict__ out, int N, int K,
                                                           int G) {
  const int kb_n = (K + 127) >> 7, kb = blockIdx.x % kb_n, tile = blockIdx.x / kb_n;
  const int gn = 128 / G;
  const uint32_t* w = W + static_cast<long>(blockIdx.x) * 256;
  // thread: row c, columns 8 u .. + 7 of the block
  const int c = threadIdx.x >> 4, u = threadIdx.x & 15, j = u >> 2, g = u & 3;
  const int n = 16 * tile + c, k = 128 * kb + 8 * u;
  if (n >= N || k >= K) return;
  const uint32_t v = w[(16 * g + c) * 4 + j];
  const long at = ((static_cast<long>(tile) * kb_n + kb) * gn + 8 * u / G) * 16 + c;
  const float s = to_f32(scale[at]), z = zero ? to_f32(zero[at]) : 8.0f;
  bf16* o = out + static_cast<long>(n) * K + k;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (k + i < K) o[i] = from_f32<bf16>(s * (static_cast<float>((v >> (4 * i)) & 15u) - z));
}

template <int CT, int G, bool Z, int R, int NW>
void int4_go(const void* x, const void* xscale, Int4Segs& sg, int M, int K, int ldx, hipStream_t s) {
  sg.blk0[0] = 0;
  for (int i = 0; i < kInt4Segs; ++i)
    sg.blk0[i + 1] = sg.blk0[i] + (i < sg.nseg ? ((sg.N[i] + 15) / 16 + R - 1) / R : 0);
  hipLaunchKernelGGL((int4_linear_kernel<CT, G, Z, R, NW>), dim3(sg.blk0[sg.nseg]), dim3(64 * NW), 0,
                     s, static_cast<const bf16*>(x), static_cast<const bf16*>(xscale), sg, M, K, ldx);
}

template <int CT, int G, bool Z, int KW>
void int4_stream(const void* x, const void* xscale, Int4Segs& sg, int M, int K, int ldx, hipStream_t s) {
  sg.blk0[0] = 0;
  for (int i = 0; i < kInt4Segs; ++i)
    sg.blk0[i + 1] = sg.blk0[i] + (i < sg.nseg ? (sg.N[i] + 15) / 16 : 0);
  const int parts = (M + 16 * CT - 1) / (16 * CT);
  // one workgroup a CU where its registers leave room for no second one (KW = 4),
  // else two (1024 -> 32000, 4 rows: 8.3 and 6.8 us; 4096 -> 32000: 15.7 and 18.9)
  const int grid = std::min(sg.blk0[kInt4Segs], (KW == 4 ? 256 : 512) / parts);
  hipLaunchKernelGGL((int4_stream_kernel<CT, G, Z, KW>), dim3(grid, parts), dim3(512), 0, s,
                     static_cast<const bf16*>(x), static_cast<const bf16*>(xscale), sg, M, K, ldx);
}

// By K and the group, in us, by tiles and streamed.  Up to 2048 columns the stream: 1024
// -> 32000, 4 rows 8.1, 6.8; 1024 -> 1024, 1 row 3.3, 2.9; 1024 -> 4384, 4 rows,
// group 64, 3.8, 4.0.  Up to 4096 too, where group 128 gains at whole K (4096 -> 4096, 1
// row 6.8, 5.2; 4096 -> 32000, 1 row 17.2, 15.7, 32 rows 31.3, 21.3, 64 rows, in two
// parts that each read the weights, 47.6, 34.5) and loses where waves have no block
// (2560 -> 32000, 1 row 12.7, 15.2; 32 rows 22.6, 20.6).  Group 64 holds twice the
// factors and spills up to 19 registers there: 4096 -> 4096, 1 row 7.3, 6.1; 4096 ->
// 32000, 1 row 18.5, 19.1, 64 rows 51, 63; 2176 -> 32000, 1 row 12.2, 18.4.
template <int G, bool Z>
void int4_rows(const void* x, const void* xscale, Int4Segs& sg, int M, int K, int ldx, hipStream_t s) {
  const int kb = (K + 127) / 128;   // (int4_streams)
  auto stream = [&](auto kw) {
    constexpr int KW = decltype(kw)::value;
    M <= 16 ? int4_stream<1, G, Z, KW>(x, xscale, sg, M, K, ldx, s)
            : int4_stream<2, G, Z, KW>(x, xscale, sg, M, K, ldx, s);
  };
  if (kb <= 8) stream(std::integral_constant<int, 1>{});
  else if (kb <= 16) stream(std::integral_constant<int, 2>{});
  else if (kb <= 32 && G > 32) stream(std::integral_constant<int, (G > 32 ? 4 : 2)>{});
  else if (M <= 16) int4_go<1, G, Z, 2, 8>(x, xscale, sg, M, K, ldx, s);
  else if (M <= 32) int4_go<2, G, Z, 2, 8>(x, xscale, sg, M, K, ldx, s);
  else int4_go<4, G, Z, 2, 8>(x, xscale, sg, M, K, ldx, s);
}

// whether int4_rows streams the tiles past x, else it goes tile by tile
bool int4_streams(int K, int G) { return K <= (G > 32 ? 4096 : 2048); }
bool int4_group_ok(int G) { return G == 32 || G == 64 || G == 128; }

}  // namespace
}  // namespace sa

extern "C" int sa_int4_linear_bf16(const void* x, const void* xscale, int M, int K, int ldx,
                                   int group, int nseg, const int64_t* matrices, void* stream) {
  const char* who = "sa_int4_linear_bf16";
  SA_CHECK_ARG(M >= 1 && M <= 64 && K > 0 && K <= (1 << 22), "%s: M %d must be 1..64 and K %d 1..2^22",
               who, M, K);
  SA_CHECK_ARG(ldx >= K && ldx <= (1 << 23), "%s: row stride %d must be at least K %d", who, ldx, K);
  SA_CHECK_ARG(sa::int4_group_ok(group), "%s: group %d not in {32, 64, 128}", who, group);
  SA_CHECK_ARG(nseg >= 1 && nseg <= sa::kInt4Segs, "%s: %d weight matrices, 1..%d allowed", who, nseg,
               sa::kInt4Segs);
  SA_CHECK_ARG(x && matrices, "%s: null pointer", who);
  SA_CHECK_ARG(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(xscale)) & 1) == 0,
               "%s: x and xscale are not aligned to their type", who);
  sa::Int4Segs sg{};
  sg.nseg = nseg;
  const bool z = matrices[2] != 0;
  // tile by tile a workgroup of 512 threads takes two (2^32 threads a grid)
  const long max_tiles = sa::int4_streams(K, group) ? 1L << 27 : (1L << 24) - 2 * sa::kInt4Segs;
  long tiles = 0;
  for (int i = 0; i < nseg; ++i) {
    const int64_t* m = matrices + 6 * i;   // packed, scales, zeros, bias, y, N
    SA_CHECK_ARG(m[0] && m[1] && m[4] && m[5] > 0 && m[5] <= (1L << 30),
                 "%s: weight matrix %d: null pointer or N %ld", who, i, static_cast<long>(m[5]));
    SA_CHECK_ARG((m[2] != 0) == z, "%s: zero points for all weight matrices or for none", who);
    SA_CHECK_ARG((m[0] & 15) == 0 && ((m[1] | m[2]) & 7) == 0, "%s: weight matrix %d is not aligned", who, i);
    tiles += (m[5] + 15) / 16;
    SA_CHECK_ARG(tiles < max_tiles, "%s: too many columns", who);
    sg.W[i] = reinterpret_cast<const uint4*>(m[0]);
    sg.scale[i] = reinterpret_cast<const sa::bf16*>(m[1]);
    sg.zero[i] = reinterpret_cast<const sa::bf16*>(m[2]);
    sg.bias[i] = reinterpret_cast<const sa::bf16*>(m[3]);
    sg.y[i] = reinterpret_cast<sa::bf16*>(m[4]);
    sg.N[i] = static_cast<int>(m[5]);
  }
  hipStream_t s = static_cast<hipStream_t>(stream);
  sa::ProfScope prof_("int4_linear", s);
  auto go = [&](auto zc) {
    constexpr bool Z = decltype(zc)::value;
    if (group == 32) sa::int4_rows<32, Z>(x, xscale, sg, M, K, ldx, s);
    else if (group == 64) sa::int4_rows<64, Z>(x, xscale, sg, M, K, ldx, s);
    else sa::int4_rows<128, Z>(x, xscale, sg, M, K, ldx, s);
  };
  z ? go(std::integral_constant<bool, true>{}) : go(std::integral_constant<bool, false>{});
  SA_CHECK_LAUNCH(who);
  return 0;
}

extern "C" int sa_int4_dequant_bf16(const void* packed, const void* scales, const void* zeros, int N,
                                    int K, int group, void* out, void* stream) {
  const char* who = "sa_int4_dequant_bf16";
  SA_CHECK_ARG(N > 0 && K > 0 && sa::int4_group_ok(group), "%s: bad sizes N=%d K=%d group=%d", who, N, K,
               group);
  SA_CHECK_ARG(packed && scales && out, "%s: null pointer", who);
  SA_CHECK_ARG((reinterpret_cast<uintptr_t>(packed) & 3) == 0, "%s: packed weights are not aligned", who);
  const long blocks = ((N + 15L) / 16) * ((K + 127L) / 128);
  SA_CHECK_ARG(blocks < (1L << 24), "%s: weights too large", who);   // (2^32 threads a grid)
  hipStream_t s = static_cast<hipStream_t>(stream);
  sa::ProfScope prof_("int4_dequant", s);
  hipLaunchKernelGGL(sa::int4_dequant_kernel, dim3(blocks), dim3(256), 0, s,
                     static_cast<const uint32_t*>(packed), static_cast<const sa::bf16*>(scales),
                     static_cast<const sa::bf16*>(zeros), static_cast<sa::bf16*>(out), N, K, group);
  SA_CHECK_LAUNCH("int4_dequant");
  return 0;
}
