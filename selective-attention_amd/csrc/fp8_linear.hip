// Linear layers in 8 bits with block scales (gfx950).
//
//   y[m, n] = sum_b 2^(ex[m, b] + ew[n / 128, b]) sum_{k in b} cx[m, k] cw[n, k] + bias[n]
//
// cx, cw e4m3 codes, b blocks of 128 columns, ex and ew the exponents of the
// rows' and the weight's scales (e8m0 bytes, fp8_rows.hip).  The matrix cores take
// both scales with the operands (one byte a lane for its 32 columns), so the sums
// over all blocks stay in one fp32 accumulator and the scales cost nothing.  They
// take the products of 8 columns together, aligned to the largest exponent and cut
// below 2^-13 of it (found by products of powers of two); those sums are added in
// fp32.  A result is so off by at most 7 2^-13 sum |x w| before its rounding to bf16,
// for random numbers by 2^-18 to 2^-20 of it, far below that rounding; the form
// without the cut, bf16 operands, has half the rate.
//
// Three kernels by size (kFp8Shapes): few rows, where the weights' stream and its
// latency count; a ring of half-steps for what does not fill the card with large tiles;
// and those.
//
// Packed weights: tiles of 16 rows and 128 columns, (N / 16, K / 128, 8, 16, 16)
// bytes: in a tile, 16 columns of its 16 rows after each other, so that 16 lanes
// read 256 bytes in a row both from memory and from LDS.  N and K are padded with
// zeros to whole tiles.  Scales: (N / 128, 4 ceil(K / 512)) bytes.
#include "fp8.h"
#include "prof.h"

#include <algorithm>
#include <type_traits>

namespace sa {
namespace {

constexpr int kFp8Segs = 4;
struct Fp8Segs {
  const uint8_t* W[kFp8Segs];
  const uint8_t* scale[kFp8Segs];
  const bf16* bias[kFp8Segs];
  bf16* y[kFp8Segs];
  int N[kFp8Segs];
  int blk0[kFp8Segs + 1];
  int nseg;
  int stream;   // the weights pass the caches by
};

typedef int v8i __attribute__((ext_vector_type(8)));
__device__ __forceinline__ v8i join16(const uint4& a, const uint4& b) {
  return v8i{static_cast<int>(a.x), static_cast<int>(a.y), static_cast<int>(a.z), static_cast<int>(a.w),
             static_cast<int>(b.x), static_cast<int>(b.y), static_cast<int>(b.z), static_cast<int>(b.w)};
}
// c += A B, both e4m3, 16 x 16 x 128; the scale is the low byte of sa, sb
__device__ __forceinline__ v4f mfma_fp8(const v8i& a, const v8i& b, const v4f& c, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, static_cast<int>(sa), 0,
                                                          static_cast<int>(sb));
}

// A workgroup of NW waves computes R tiles of 16 columns of y for 16 CT rows of x;
// the waves take the blocks of K in turn and their sums meet in LDS.  Operands go
// from memory to registers, the next block's while this one's are multiplied: no wave
// has what another needs.  Lane 16 g + c holds columns 16 g .. + 15 and 64 + 16 g .. of a
// block, of row c.
// X: the rows are codes with scales (kCodes), or bfloat16 that each wave rounds for
// itself, block by block (kBf16; kGated: times the gate): the four lanes of a row have
// a block's columns between them, so its scale costs two lane exchanges, and up to 16
// rows save the launch that would make the codes (4 rows, 1024 -> 4384: 17.4 us a call
// with it).
enum { kCodes = 0, kBf16 = 1, kGated = 2 };
struct Fp8X {
  const void *x, *other;   // codes and scales, or rows and gate
  int64_t ldx, ldg;        // of rows in bfloat16
  int K;
};
// sixteen columns of a row from k on, those at or behind K as 0 (pieces of eight at any
// address, the row's last by elements)
typedef uint32_t v4u_any __attribute__((ext_vector_type(4), aligned(2)));
__device__ __forceinline__ void load16(uint4 (&q)[2], const bf16* row, int k, int K) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int at = k + 8 * i;
    q[i] = uint4{0u, 0u, 0u, 0u};
    if (at + 8 <= K) {
      q[i] = __builtin_bit_cast(uint4, *reinterpret_cast<const v4u_any*>(row + at));
    } else if (at < K) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t lo = at + 2 * e < K ? row[at + 2 * e].x : 0u, hi = at + 2 * e + 1 < K ? row[at + 2 * e + 1].x : 0u;
        w[e] = lo | hi << 16;
      }
      q[i] = uint4{w[0], w[1], w[2], w[3]};
    }
  }
}
__device__ __forceinline__ uint32_t word_of(const uint4 (&q)[2], int i) {
  const uint4& u = q[i >> 2];
  return (i & 3) == 0 ? u.x : (i & 3) == 1 ? u.y : (i & 3) == 2 ? u.z : u.w;
}
__device__ __forceinline__ void widen16(float* v, const uint4 (&q)[2]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[2 * i] = bf16lo_to_f32(word_of(q, i));
    v[2 * i + 1] = bf16hi_to_f32(word_of(q, i));
  }
}
template <int CT, int R, int NW, int X>
__global__ __launch_bounds__(64 * NW) void fp8_few_kernel(const Fp8X in, const Fp8Segs sg, int M, int kb_n) {
  __shared__ float part[NW * R * CT * 256];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6, c = lane & 15, g = lane >> 4;
  const int across = sg.blk0[kFp8Segs];   // workgroups a row of tiles
  const int bid = blockIdx.x % across, m0 = blockIdx.x / across * 16 * CT;
  int seg = 0;
#pragma unroll
  for (int i = 1; i < kFp8Segs; ++i) seg += (i < sg.nseg && bid >= sg.blk0[i]) ? 1 : 0;
  const int N = sg.N[seg], tiles = (N + 15) >> 4, words = (kb_n + 3) >> 2;
  const int t0 = (bid - sg.blk0[seg]) * R;
  // (rows and tiles behind the last are the last again, not stored)
  const uint4* wp[R];
  const uint4* xp[CT];
  const uint8_t* sxp[CT];
  const bf16 *xr[CT], *gr[CT];
#pragma unroll
  for (int r = 0; r < R; ++r)
    wp[r] = reinterpret_cast<const uint4*>(sg.W[seg] + static_cast<long>(min(t0 + r, tiles - 1)) * kb_n * 2048) + lane;
#pragma unroll
  for (int t = 0; t < CT; ++t) {
    const long row = min(m0 + 16 * t + c, M - 1);
    if constexpr (X == kCodes) {
      xp[t] = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(in.x) + row * kb_n * 128) + g;
      sxp[t] = static_cast<const uint8_t*>(in.other) + row * 4 * words;
    } else {
      xr[t] = static_cast<const bf16*>(in.x) + row * in.ldx;
      if constexpr (X == kGated) gr[t] = static_cast<const bf16*>(in.other) + row * in.ldg;
    }
  }
  const uint8_t* swp[R];
#pragma unroll
  for (int r = 0; r < R; ++r) swp[r] = sg.scale[seg] + static_cast<long>(min(t0 + r, tiles - 1) >> 3) * 4 * words;

  struct Block {
    uint4 w[R][2], x[CT][X == kCodes ? 1 : 2][2], gate[X == kGated ? CT : 1][2][2];
    uint32_t sw[R], sx[CT];
  };
  auto load = [&](int kb, Block& q) __attribute__((always_inline)) {
    if (sg.stream) {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          q.w[r][i] = __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const v4f*>(wp[r] + kb * 128 + 64 * i)));
    } else {
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < 2; ++i) q.w[r][i] = wp[r][kb * 128 + 64 * i];
    }
#pragma unroll
    for (int r = 0; r < R; ++r) q.sw[r] = swp[r][kb];
#pragma unroll
    for (int t = 0; t < CT; ++t) {
      if constexpr (X == kCodes) {
        q.x[t][0][0] = xp[t][kb * 8];
        q.x[t][0][1] = xp[t][kb * 8 + 4];
        q.sx[t] = sxp[t][kb];
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          load16(q.x[t][i], xr[t], 128 * kb + 64 * i + 16 * g, in.K);
          if constexpr (X == kGated) load16(q.gate[t][i], gr[t], 128 * kb + 64 * i + 16 * g, in.K);
        }
      }
    }
  };
  v4f acc[R][CT];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < CT; ++t) acc[r][t] = v4f{0.f, 0.f, 0.f, 0.f};
  auto multiply = [&](const Block& q) __attribute__((always_inline)) {
#pragma unroll
    for (int t = 0; t < CT; ++t) {
      v8i xf;
      uint32_t sx;
      if constexpr (X == kCodes) {
        xf = join16(q.x[t][0][0], q.x[t][0][1]);
        sx = q.sx[t];
      } else {
        // (infinities apart, the codes come straight from the bf16 words, or the products)
        float v[32], top = 0.0f;
#pragma unroll
        for (int i = 0; i < 2; ++i) widen16(v + 16 * i, q.x[t][i]);
        if constexpr (X == kGated) {
          float f[32];
#pragma unroll
          for (int i = 0; i < 2; ++i) widen16(f + 16 * i, q.gate[t][i]);
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] *= f[i];   // (exact but for those below fp32's normal numbers)
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) top = fmaxf(top, fabsf(v[i]));   // (a NaN is passed over)
        if constexpr (X == kGated) {
          if (__any(top < 0x1p-100f && top != 0.0f)) {
            top = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              uint32_t a = word_of(q.x[t][i >> 3], i & 7), b = word_of(q.gate[t][i >> 3], i & 7);
              asm volatile("" : "+v"(a), "+v"(b));   // (widened anew: the first copies would stay in registers)
              v[2 * i] = to_odd(static_cast<double>(bf16lo_to_f32(a)) * bf16lo_to_f32(b));
              v[2 * i + 1] = to_odd(static_cast<double>(bf16hi_to_f32(a)) * bf16hi_to_f32(b));
              top = fmaxf(top, fmaxf(fabsf(v[2 * i]), fabsf(v[2 * i + 1])));
            }
          }
        }
        const bool rare = __any(top == __builtin_inff());
        if (rare) {
          top = 0.0f;
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            v[i] = no_infinity(v[i]);
            top = fmaxf(top, fabsf(v[i]));
          }
        }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        sx = scale_byte(fmaxf(top, __shfl_xor(top, 32, 64)));
        const float scale = scale_value(sx);
        if (X == kGated || rare) {
#pragma unroll
          for (int i = 0; i < 8; ++i) xf[i] = static_cast<int>(encode4(v + 4 * i, scale));
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint4& u = q.x[t][i >> 1][i & 1];
            xf[2 * i] = static_cast<int>(encode4(u.x, u.y, scale));
            xf[2 * i + 1] = static_cast<int>(encode4(u.z, u.w, scale));
          }
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) acc[r][t] = mfma_fp8(join16(q.w[r][0], q.w[r][1]), xf, acc[r][t], q.sw[r], sx);
    }
  };
  // (two copies of the body, so that no register of a load in flight is moved)
  Block q0, q1;
  int kb = wid;
  if (kb < kb_n) load(kb, q0);
  while (kb < kb_n) {
    if (kb + NW < kb_n) load(kb + NW, q1);
    multiply(q0);
    kb += NW;
    if (kb >= kb_n) break;
    if (kb + NW < kb_n) load(kb + NW, q0);
    multiply(q1);
    kb += NW;
  }
  // lane (c, g) holds columns 4 g + e of the tile for row 16 t + c of x
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int t = 0; t < CT; ++t)
      *reinterpret_cast<float4*>(part + ((wid * CT + t) * 16 + c) * 16 * R + 16 * r + 4 * g) =
          make_float4(acc[r][t][0], acc[r][t][1], acc[r][t][2], acc[r][t][3]);
  __syncthreads();
  const bf16* bias = sg.bias[seg];
  bf16* y = sg.y[seg];
  for (int e = tid; e < R * CT * 256; e += 64 * NW) {
    const int row = m0 + e / (16 * R), n = 16 * t0 + e % (16 * R);
    float v = 0.0f;
#pragma unroll
    for (int i = 0; i < NW; ++i) v += part[i * R * CT * 256 + e];
    if (row < M && n < N) y[static_cast<long>(row) * N + n] = from_f32<bf16>(v + (bias ? to_f32(bias[n]) : 0.0f));
  }
}

typedef float v16f __attribute__((ext_vector_type(16)));
// c += A B, both e4m3, 32 x 32 x 64
__device__ __forceinline__ v16f mfma_fp8(const v8i& a, const v8i& b, const v16f& c, uint32_t sa, uint32_t sb) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, static_cast<int>(sa), 0,
                                                         static_cast<int>(sb));
}
__device__ __forceinline__ v8i lds_frag(const uint8_t* p, const uint8_t* q) {
  return join16(*reinterpret_cast<const uint4*>(p), *reinterpret_cast<const uint4*>(q));
}
// (memory is not moved past it)
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
using yes = std::integral_constant<bool, true>;
using no = std::integral_constant<bool, false>;

// What a workgroup of a tile kernel computes: columns n0 .. of matrix seg for rows m0 ..
struct Fp8Tile {
  int seg, n0, m0;
};
// Tiles in the order of the XCDs, a part of the list each, so that an L2 serves
// neighbours; in it, `high` rows of tiles at a time
template <int BN, int BM>
__device__ __forceinline__ Fp8Tile tile_of(const Fp8Segs& sg, int mtiles) {
  const int ntiles = sg.blk0[kFp8Segs], total = ntiles * mtiles, xcd = blockIdx.x & 7;
  const int id = xcd * (total >> 3) + min(xcd, total & 7) + (blockIdx.x >> 3);
  const int band = id / (4 * ntiles), left = id - band * 4 * ntiles, high = min(4, mtiles - 4 * band);
  const int nt = left / high;
  Fp8Tile t{0, 0, (4 * band + left % high) * BM};
#pragma unroll
  for (int i = 1; i < kFp8Segs; ++i) t.seg += (i < sg.nseg && nt >= sg.blk0[i]) ? 1 : 0;
  t.n0 = (nt - sg.blk0[t.seg]) * BN;
  return t;
}

// The scales of a wave's 32 SN columns and 32 SM rows, a word for four blocks: the
// rows' a lane each, the weight's one for the wave (columns of one block of 128)
template <int SM>
struct Fp8Scales {
  const uint32_t *w, *x;
  uint32_t at[SM], sx[SM], nx[SM], sw, nw;
  int words;
  __device__ __forceinline__ Fp8Scales(const Fp8Segs& sg, const uint8_t* xs, const Fp8Tile& t, int n, int m, int M,
                                       int words_) : words(words_) {
    w = reinterpret_cast<const uint32_t*>(sg.scale[t.seg]) + static_cast<long>(min(n, sg.N[t.seg] - 1) >> 7) * words;
    x = reinterpret_cast<const uint32_t*>(xs) + static_cast<long>(t.m0) * words;
#pragma unroll
    for (int j = 0; j < SM; ++j)
      at[j] = static_cast<uint32_t>(min(m - t.m0 + 32 * j + static_cast<int>(threadIdx.x & 31), M - 1 - t.m0)) * words;
    load(0);
  }
  __device__ __forceinline__ void load(int g) {   // the next word
    nw = w[g];
#pragma unroll
    for (int j = 0; j < SM; ++j) nx[j] = x[at[j] + g];
  }
  __device__ __forceinline__ void take() {
    sw = nw;
#pragma unroll
    for (int j = 0; j < SM; ++j) sx[j] = nx[j];
  }
  // from block t to the next: the low byte is block t + 1's
  __device__ __forceinline__ void step(int t) {
    if ((t & 3) == 3) return take();
    sw >>= 8;
#pragma unroll
    for (int j = 0; j < SM; ++j) sx[j] >>= 8;
  }
  // a word two blocks ahead of its use
  __device__ __forceinline__ void ahead(int t) {
    if ((t & 3) == 1) load(min((t >> 2) + 1, words - 1));
  }
};

// The wave's 32 SM rows and 32 SN columns of y, through its own part of LDS (32 rows
// of kCols columns at a time) so that they leave as whole pieces of 2 kCols bytes.  They
// pass the caches by: nothing here reads them again, and the next tiles' operands
// stay (32768 rows, 1024 -> 4096: 165 us, so 142).
typedef float v4f_any __attribute__((ext_vector_type(4), aligned(2)));   // 16 bytes at any even address
template <int SN, int SM>
struct Fp8Out {
  static constexpr int kCols = SN > 1 ? 64 : 32, kPitch = 2 * kCols + 16, kBytes = 32 * kPitch;
  static __device__ __forceinline__ void store(const v16f (&acc)[SN][SM], uint8_t* ys, const float* bias, bf16* y0,
                                               int nw, int mw, int N, int M) {
    const int lane = threadIdx.x & 63, c = lane & 31, h = lane >> 5;
    bf16* y = y0 + static_cast<long>(mw) * N + nw;
    constexpr int kSq = kCols / 32, kLanes = kCols / 8;
#pragma unroll
    for (int j = 0; j < SM; ++j)
#pragma unroll
      for (int i0 = 0; i0 < SN; i0 += kSq) {
        // lane (c, h) holds columns 8 q + 4 h + e of square i for row c
#pragma unroll
        for (int i = 0; i < kSq; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const v16f& a = acc[i0 + i][j];
            const float4 b = *reinterpret_cast<const float4*>(bias + 32 * (i0 + i) + 8 * q + 4 * h);
            *reinterpret_cast<uint2*>(ys + c * kPitch + (32 * i + 8 * q + 4 * h) * 2) =
                uint2{pack_bf16x2(a[4 * q] + b.x, a[4 * q + 1] + b.y), pack_bf16x2(a[4 * q + 2] + b.z, a[4 * q + 3] + b.w)};
          }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int r = 0; r < 32; r += 64 / kLanes) {
          const int row = r + lane / kLanes, n = 32 * i0 + 8 * (lane % kLanes), left = mw + 32 * j + row < M ? N - nw - n : 0;
          bf16* to = y + static_cast<long>(32 * j + row) * N + n;
          const uint8_t* from = ys + row * kPitch + 16 * (lane % kLanes);
          if (left >= 8) {
            __builtin_nontemporal_store(*reinterpret_cast<const v4f*>(from), reinterpret_cast<v4f_any*>(to));
          } else {   // the matrix's last columns
#pragma unroll 1
            for (int e = 0; e < left; ++e) to[e] = *reinterpret_cast<const bf16*>(from + 2 * e);
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
  }
};

// A workgroup of four waves (2 by 2) computes 64 SN columns of y for 64 SM rows of x;
// a wave SN by SM squares of 32 (W as the first operand, so that a lane holds four
// neighbouring columns of one row).  A step is one block of 128 columns of K, in LDS in
// two stages that DMA fills: W as it is packed, x as rows of 128 bytes whose pieces of
// 16 are permuted by row (piece p of row r at p ^ (r / 2 & 7)), so that sixteen lanes
// read all banks.  Operands are held for half a step (64 columns): while the matrix
// cores take one half, the next is read, also over the steps' border, so that a step
// needs one barrier, in its middle: there this step's stage has been read by all and
// the next one has landed.  For large products, 256 by 256 with one wave a SIMD (its
// sums fill half of the registers): of all shapes it reads LDS the least.  8192 x 8192 x
// 8192 412 us, 2670 TFLOP/s, with the matrix cores busy in 73 % of the cycles at 1.6 to
// 1.75 GHz: full of such tiles the card lowers its clock, so that fewer idle cycles do
// not end it sooner (bank conflicts cut to a tenth: the same time).
template <int SN, int SM>
__global__ __launch_bounds__(256, 1) void fp8_large_kernel(const uint8_t* __restrict__ x,
                                                           const uint8_t* __restrict__ xs, const Fp8Segs sg, int M,
                                                           int kb_n, int mtiles) {
  constexpr int BN = 64 * SN, BM = 64 * SM, kW = BN * 128, kStage = (BN + BM) * 128;
  using Out = Fp8Out<SN, SM>;
  static_assert(4 * Out::kBytes <= 2 * kStage, "y fits the stages");
  __shared__ __align__(16) uint8_t smem[2 * kStage + 4 * BN];
  float* bias_lds = reinterpret_cast<float*>(smem + 2 * kStage);
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, h = lane >> 5;
  const int wid = __builtin_amdgcn_readfirstlane(tid >> 6), wn = wid & 1, wm = wid >> 1;
  const Fp8Tile tile = tile_of<BN, BM>(sg, mtiles);
  const int N = sg.N[tile.seg], n0 = tile.n0, m0 = tile.m0, nw = n0 + wn * 32 * SN, mw = m0 + wm * 32 * SM;
  const bf16* bias = sg.bias[tile.seg];
  if (tid < BN) bias_lds[tid] = bias && n0 + tid < N ? to_f32(bias[n0 + tid]) : 0.0f;

  // DMA: 1 KB an instruction; a wave takes SN * 2 of W (a tile's half each) and SM * 2 of x
  // (eight rows); what lies behind the last tile or row is the last again and not stored
  const uint32_t ls = lds_addr(smem);
  const uint8_t* wbase = sg.W[tile.seg] + static_cast<long>(n0 >> 4) * kb_n * 2048;
  const uint8_t* xbase = x + static_cast<long>(m0) * kb_n * 128;
  uint32_t woff[2 * SN], xoff[2 * SM];
#pragma unroll
  for (int i = 0; i < 2 * SN; ++i) {
    const int q = wid * 2 * SN + i, t = min(q >> 1, ((N + 15) >> 4) - 1 - (n0 >> 4));
    woff[i] = static_cast<uint32_t>(t) * kb_n * 2048 + (q & 1) * 1024 + lane * 16;
  }
#pragma unroll
  for (int i = 0; i < 2 * SM; ++i) {
    const int r = min((wid * 2 * SM + i) * 8 + (lane >> 3), M - 1 - m0);
    xoff[i] = static_cast<uint32_t>(r) * kb_n * 128 + ((lane & 7) ^ ((lane >> 4) + 4 * (i & 1))) * 16;
  }
  auto dma = [&](int i, int t, uint32_t stage) __attribute__((always_inline)) {
    if (i < 2 * SN) dma_lds16(wbase + static_cast<long>(t) * 2048, woff[i], stage + ((wid * 2 * SN + i) << 10));
    else if (i < 2 * (SN + SM))
      dma_lds16(xbase + static_cast<long>(t) * 128, xoff[i - 2 * SN], stage + kW + ((wid * 2 * SM + i - 2 * SN) << 10));
  };
  auto dma_all = [&](int t, uint32_t stage) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 2 * (SN + SM); ++i) dma(i, t, stage);
  };

  // operands' places in a stage: piece 4 half + 2 h + i of a row
  const int wa = wn * SN * 4096 + (c >> 4) * 2048 + h * 512 + (c & 15) * 16;
  int xa[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    xa[i] = kW + wm * SM * 4096 + c * 128 + ((((i >> 1) * 4 + 2 * h + (i & 1)) ^ ((c >> 1) & 7)) * 16);
  v8i fw[2][SN], fx[2][SM];
  // operand r in the order in which the products need them: one of W, those of x, the rest of W
  auto read_frag = [&](int half, int r, int stage) __attribute__((always_inline)) {
    if (r == 0 || (r > SM && r < SN + SM)) {
      const int s = r == 0 ? 0 : r - SM;
      const uint8_t* p = smem + stage + wa + s * 4096 + half * 1024;
      fw[half][s] = lds_frag(p, p + 256);
    } else if (r <= SM) {
      const uint8_t* p = smem + stage + (r - 1) * 4096;
      fx[half][r - 1] = lds_frag(p + xa[2 * half], p + xa[2 * half + 1]);
    }
  };
  constexpr int kSlots = SN * SM, kReads = (SN + SM + kSlots - 1) / kSlots, kDma = (2 * (SN + SM) + kSlots - 1) / kSlots;

  v16f acc[SN][SM] = {};
  dma_all(0, ls);
  Fp8Scales<SM> sc(sg, xs, tile, nw, mw, M, (kb_n + 3) >> 2);
  __builtin_amdgcn_s_waitcnt(vm_lgkm_wait<0>());
  lds_barrier();
  sc.take();
  if (kb_n > 1) dma_all(1, ls + kStage);
#pragma unroll
  for (int r = 0; r < SN + SM; ++r) read_frag(0, r, 0);

  // step t: a step t + 1 follows (NEXT), a step t + 2 (MORE)
  auto step = [&](int t, auto next, auto more) __attribute__((always_inline)) {
    constexpr bool NEXT = decltype(next)::value, MORE = decltype(more)::value;
    const int cur = (t & 1) * kStage, oth = kStage - cur;
    if (NEXT) sc.ahead(t);
    // (the order is kept as written: reads and DMA go out between the products)
#pragma unroll
    for (int k = 0; k < kSlots; ++k) {
      const int i = k / SM, j = k % SM;
      acc[i][j] = mfma_fp8(fw[0][i], fx[0][j], acc[i][j], sc.sw, sc.sx[j]);
#pragma unroll
      for (int r = k * kReads; r < (k + 1) * kReads; ++r) read_frag(1, r, cur);
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (NEXT) {
      __builtin_amdgcn_s_waitcnt(vm_lgkm_wait<0>());
      lds_barrier();   // this stage is read by all, the next one has landed
    }
#pragma unroll
    for (int k = 0; k < kSlots; ++k) {
      const int i = k / SM, j = k % SM;
      acc[i][j] = mfma_fp8(fw[1][i], fx[1][j], acc[i][j], sc.sw, sc.sx[j]);
      if constexpr (NEXT) {
#pragma unroll
        for (int r = k * kReads; r < (k + 1) * kReads; ++r) read_frag(0, r, oth);
      }
      if constexpr (MORE) {
#pragma unroll
        for (int d = k * kDma; d < (k + 1) * kDma; ++d) dma(d, t + 2, ls + cur);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (NEXT) sc.step(t);
  };
  int t = 0;
  for (; t + 2 < kb_n; ++t) step(t, yes{}, yes{});
  if (t + 1 < kb_n) step(t++, yes{}, no{});
  step(t, no{}, no{});

  __builtin_amdgcn_s_waitcnt(kLgkmWait0);
  lds_barrier();
  Out::store(acc, smem + wid * Out::kBytes, bias_lds + wn * 32 * SN, sg.y[tile.seg], nw, mw, N, M);
}

// keeps a product where it is written, between the reads and DMA around it
__device__ __forceinline__ void pin(v16f& c) { asm volatile("" : "+a"(c)::"memory"); }

// The same for fewer rows and columns than fill the card with such tiles.  A step is
// half a block, in a ring of R stages, R - 1 on their way while one is multiplied: a
// tile alone on its CU waits for nothing but memory's first answer if the ring is deep,
// several on a CU cover each other and leave room for fewer stages.
// x lies in rows of 64 bytes, piece p of row r at p ^ (r / 4 & 3).  The scales' words come
// with every eighth half-step, into two places in turn (a load into a register would make
// the compiler wait for all DMA before its use; with every half-step they took more of
// the cache's time than the operands, each row's word being a line of its own: 1000 rows,
// 11008 -> 4096 59 us, so 47).
// KS = 2: eight waves, a ring and one half of K for each four, whose sums meet in LDS:
// small tiles wait less than their operands take (512 rows, 4096 -> 1024: 12.4 us, so 11.1;
// below eight blocks a half is too short, 512 -> 1024: 4.5, so 4.9).
template <int SN, int SM, int R, int OCC, int KS, bool NT>
__global__ __launch_bounds__(256 * KS, OCC * KS) void fp8_ring_kernel(const uint8_t* __restrict__ x,
                                                                      const uint8_t* __restrict__ xs, const Fp8Segs sg,
                                                                      int M, int kb_n, int mtiles) {
  constexpr int BN = 64 * SN, BM = 64 * SM, kW = BN * 64, kStage = (BN + BM) * 64;
  constexpr int kScales = R * kStage, kRing = kScales + 2048, kSums = SN * SM * 4096;   // (a wave's sums, in bytes)
  constexpr int kParts = (BN + BM) / 16, kDmas = (kParts + 3) / 4;   // DMA instructions of a stage, and of a wave
  static_assert(BM <= 128 && BN <= 256, "a word's scales: two waves' rows, one's columns");
  static_assert(R >= 3 && R <= 6, "landed knows them; the word after the next comes when this one's has been read");
  static_assert((R - 1) * kDmas + 1 < 63, "vmcnt counts them");
  using Out = Fp8Out<SN, SM>;
  static_assert(4 * Out::kBytes <= R * kStage, "y fits the stages");
  static_assert(KS == 1 || (KS == 2 && 4 * kSums <= KS * kRing && Out::kBytes <= kSums), "sums and y fit the rings");
  __shared__ __align__(16) uint8_t smem[KS * kRing + 4 * BN];
  float* bias_lds = reinterpret_cast<float*>(smem + KS * kRing);
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), part = wave >> 2, wid = wave & 3, wn = wid & 1, wm = wid >> 1;
  const Fp8Tile tile = tile_of<BN, BM>(sg, mtiles);
  const int N = sg.N[tile.seg], n0 = tile.n0, m0 = tile.m0, nw = n0 + wn * 32 * SN, mw = m0 + wm * 32 * SM;
  const bf16* bias = sg.bias[tile.seg];
  if (tid < BN) bias_lds[tid] = bias && n0 + tid < N ? to_f32(bias[n0 + tid]) : 0.0f;

  // the half-steps u0 to U - 1 of this part of the waves
  const int most = 2 * ((kb_n + KS - 1) / KS), u0 = part * most, U = min(u0 + most, 2 * kb_n);
  // piece q of a stage: half a tile of W, or sixteen rows of x; wave w takes w, w + 4, ..
  // (a piece too many is the last again, at the same place)
  uint8_t* ring = smem + part * kRing;
  const uint32_t ls = lds_addr(ring);
  const uint8_t* d_w = sg.W[tile.seg] + static_cast<long>(n0 >> 4) * kb_n * 2048;
  const uint8_t* d_x = x + static_cast<long>(m0) * kb_n * 128;
  uint32_t off[kDmas], s_off;
#pragma unroll
  for (int i = 0; i < kDmas; ++i) {
    const int q = min(wid + 4 * i, kParts - 1);
    off[i] = q < BN / 16 ? static_cast<uint32_t>(min(q, ((N + 15) >> 4) - 1 - (n0 >> 4))) * kb_n * 2048 + lane * 16
                         : static_cast<uint32_t>(min((q - BN / 16) * 16 + (lane >> 2), M - 1 - m0)) * kb_n * 128 +
                               ((lane & 3) ^ (lane >> 4)) * 16;
  }
  // words of scales: waves 0 and 1 of 64 rows each, 2 and 3 of the groups of 32 columns
  const int words = (kb_n + 3) >> 2;
  const uint8_t* d_s;
  if (wid < 2) {
    d_s = xs + static_cast<long>(m0) * 4 * words;
    s_off = static_cast<uint32_t>(min(64 * wid + lane, M - 1 - m0)) * 4 * words;
  } else {
    d_s = sg.scale[tile.seg] + static_cast<long>(n0 >> 7) * 4 * words;
    s_off = static_cast<uint32_t>((min(n0 + 32 * min(lane, BN / 32 - 1), N - 1) >> 7) - (n0 >> 7)) * 4 * words;
  }
  d_w += static_cast<long>(u0) * 1024;
  d_x += static_cast<long>(u0) * 64;
  int d_u = u0;
  auto word_at = [&](int u) __attribute__((always_inline)) { return ((u >> 3) & 1) * 1024; };
  auto dma = [&](int i, uint32_t stage) __attribute__((always_inline)) {
    const int q = min(wid + 4 * i, kParts - 1);
    if (i == 0 && ((d_u & 7) == 0 || (KS > 1 && d_u == u0)))
      dma_lds4(d_s + (d_u >> 3) * 4, s_off, ls + kScales + word_at(d_u) + (wid << 8));
    if (i >= kDmas) return;
    if (NT && i < BN / 64) dma_lds16_nt(d_w, off[i], stage + (q << 10));
    else dma_lds16(q < BN / 16 ? d_w : d_x, off[i], stage + (q << 10));
  };
  auto advance = [&]() __attribute__((always_inline)) {
    d_w += 1024;
    d_x += 64;
    ++d_u;
  };

  const int wa = wn * SN * 2048 + (c >> 4) * 1024 + h * 512 + (c & 15) * 16;
  int xa[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) xa[i] = kW + wm * SM * 2048 + c * 64 + (((2 * h + i) ^ ((c >> 2) & 3)) * 16);
  const int sxa = kScales + (wm * SM * 32 + c) * 4, swa = kScales + 512 + wn * SN * 4;
  v8i fw[2][SN], fx[2][SM];
  uint32_t sw[2], sx[2][SM];
  auto read_frag = [&](int half, int r, int stage, int word) __attribute__((always_inline)) {
    if (r == 0) {
      sw[half] = *reinterpret_cast<const uint32_t*>(ring + word + swa);
#pragma unroll
      for (int j = 0; j < SM; ++j) sx[half][j] = *reinterpret_cast<const uint32_t*>(ring + word + sxa + 128 * j);
    }
    if (r == 0 || (r > SM && r < SN + SM)) {
      const int s = r == 0 ? 0 : r - SM;
      const uint8_t* p = ring + stage + wa + s * 2048;
      fw[half][s] = lds_frag(p, p + 256);
    } else if (r <= SM) {
      const uint8_t* p = ring + stage + (r - 1) * 2048;
      fx[half][r - 1] = lds_frag(p + xa[0], p + xa[1]);
    }
  };
  // all but the newest n stages of DMA have landed, and the wave's reads (a scales' word
  // among the newest, not counted, lets one piece less be on its way)
  auto landed = [&](int n) __attribute__((always_inline)) {
    switch (n) {
#define SA_FP8_WAIT(k) \
  case k: \
    if constexpr (k < R - 1) __builtin_amdgcn_s_waitcnt(vm_lgkm_wait<(k < R - 1 ? k : 0) * kDmas>()); \
    break;
      SA_FP8_WAIT(1) SA_FP8_WAIT(2) SA_FP8_WAIT(3) SA_FP8_WAIT(4)
#undef SA_FP8_WAIT
      default: __builtin_amdgcn_s_waitcnt(vm_lgkm_wait<0>());
    }
  };

  const int filled = min(U - u0, R);
  v16f acc[SN][SM] = {};
  for (int s = 0; s < filled; ++s) {
#pragma unroll
    for (int i = 0; i < kDmas; ++i) dma(i, ls + s * kStage);
    advance();
  }
  landed(filled - 2);   // (at least two)
  lds_barrier();
#pragma unroll
  for (int r = 0; r < SN + SM; ++r) read_frag(0, r, 0, word_at(u0));
  __builtin_amdgcn_s_waitcnt(kLgkmWait0);
  lds_barrier();

  // half-step u on stage cur, whose operands are in registers and which all have read:
  // those of u + 1 are read, stage cur takes half-step u + R
  int cur = 0, u = u0;
  auto half_step = [&](auto half, auto more) __attribute__((always_inline)) {
    constexpr int HF = decltype(half)::value;
    constexpr bool MORE = decltype(more)::value;
    const int shift = (u >> 1 & 3) * 8;   // the block's byte
    const int word = word_at(u + 1);
    const int oth = cur == (R - 1) * kStage ? 0 : cur + kStage;
    constexpr int kSlots = SN * SM, kReads = (SN + SM + kSlots - 1) / kSlots, kPer = (kDmas + kSlots - 1) / kSlots;
#pragma unroll
    for (int k = 0; k < kSlots; ++k) {
      const int i = k / SM, j = k % SM;
      acc[i][j] = mfma_fp8(fw[HF][i], fx[HF][j], acc[i][j], sw[HF] >> shift, sx[HF][j] >> shift);
      pin(acc[i][j]);
#pragma unroll
      for (int r = k * kReads; r < (k + 1) * kReads; ++r) read_frag(HF ^ 1, r, oth, word);   // (of the last: not used)
      if constexpr (MORE) {
#pragma unroll
        for (int d = k * kPer; d < (k + 1) * kPer; ++d) dma(d, ls + cur);
      }
    }
    if constexpr (MORE) {
      advance();
      __builtin_amdgcn_s_waitcnt(vm_lgkm_wait<(R - 2) * kDmas>());
    } else {
      landed(U - 3 - u);
    }
    lds_barrier();
    cur = oth;
    ++u;
  };
  using h0 = std::integral_constant<int, 0>;
  using h1 = std::integral_constant<int, 1>;
  while (u + 1 + R < U) {
    half_step(h0{}, yes{});
    half_step(h1{}, yes{});
  }
  if (R % 2 == 1 && u + R < U) {
    half_step(h0{}, yes{});
    half_step(h1{}, no{});
  }
  while (u < U) {
    half_step(h0{}, no{});
    half_step(h1{}, no{});
  }
  if constexpr (KS > 1) {
    for (int i = U - u0; i < most; ++i) lds_barrier();   // (as many as the other part)
    float4* sums = reinterpret_cast<float4*>(smem + wid * kSums) + lane;
    if (part) {
#pragma unroll
      for (int i = 0; i < SN * SM * 4; ++i) {
        const v16f& a = acc[i / 4 / SM][i / 4 % SM];
        sums[64 * i] = make_float4(a[i % 4 * 4], a[i % 4 * 4 + 1], a[i % 4 * 4 + 2], a[i % 4 * 4 + 3]);
      }
    }
    __syncthreads();
    if (part) return;
#pragma unroll
    for (int i = 0; i < SN * SM * 4; ++i) {
      const float4 b = sums[64 * i];
      v16f& a = acc[i / 4 / SM][i / 4 % SM];
      a[i % 4 * 4] += b.x;
      a[i % 4 * 4 + 1] += b.y;
      a[i % 4 * 4 + 2] += b.z;
      a[i % 4 * 4 + 3] += b.w;
    }
  }
  Out::store(acc, smem + wid * (KS > 1 ? kSums : Out::kBytes), bias_lds + wn * 32 * SN, sg.y[tile.seg], nw, mw, N, M);
}

// the weights in bf16, (N, K) row-major; a code times its scale is a bf16 number
// (but for scales below 2^-117).  One workgroup a tile and block: 16384 x 16384 143 us,
// 5.6 TB/s (stores of single elements 497).
__global__ __launch_bounds__(128) void fp8_dequant_kernel(const uint8_t* __restrict__ W,
                                                          const uint8_t* __restrict__ scale, bf16* __restrict__ out,
                                                          int N, int K, int kb_n) {
  const int kb = blockIdx.x % kb_n, tile = blockIdx.x / kb_n;
  const int j = threadIdx.x >> 4, l = threadIdx.x & 15, half = l & 1;   // piece of 16 columns, its half
  const uint32_t byte = scale[static_cast<long>(tile >> 3) * 4 * ((kb_n + 3) >> 2) + kb];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = (l >> 1) + 8 * i, n = 16 * tile + r, k = 128 * kb + 16 * j + 8 * half;
    const uint2 q = *reinterpret_cast<const uint2*>(W + static_cast<long>(blockIdx.x) * 2048 + j * 256 + r * 16 + 8 * half);
    if (n >= N) continue;
    const uint32_t u[2] = {q.x, q.y};
    bf16* o = out + static_cast<long>(n) * K + k;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      v[e] = ldexpf(__builtin_amdgcn_cvt_f32_fp8(static_cast<int>(u[e >> 2] >> (8 * (e & 3))), 0), static_cast<int>(byte) - 127);
    if (k <= K - 8) {   // (K may be int's last)
      *reinterpret_cast<v4u_any*>(o) =
          v4u_any{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (k + e < K) o[e] = from_f32<bf16>(v[e]);
    }
  }
}

// The bias's gradient: sums over the rows of x (rows, N), in fp32.  A workgroup takes 64
// columns of `chunk` rows, eight columns a thread (128 bytes of a row, a line) and every
// 32nd row, whose sums meet in LDS; more chunks than one go to a second pass over their
// sums, in order.  32768 x 4096 46 us, 5.8 TB/s; 32768 x 1024 15.5, where 256 columns a
// workgroup and 256 chunks took 47 in the second pass; 4095 columns 112, no row on a line.
constexpr int kSumCols = 64, kSumRows = 32;
template <typename TI, typename TO>
__global__ __launch_bounds__(256) void colsum_kernel(const TI* __restrict__ x, TO* __restrict__ out, long rows, int N,
                                                     int chunk) {
  __shared__ float part[kSumRows][kSumCols];
  const int c = threadIdx.x & 7, g = threadIdx.x >> 3, n = blockIdx.x * kSumCols + 8 * c;
  const long r0 = static_cast<long>(blockIdx.y) * chunk, r1 = min(rows, r0 + chunk);
  float acc[8] = {};
  if (sizeof(TI) == 2 && n + 8 <= N) {
#pragma unroll 8
    for (long r = r0 + g; r < r1; r += kSumRows) {
      const v4u_any q = *reinterpret_cast<const v4u_any*>(x + r * N + n);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        acc[2 * i] += bf16lo_to_f32(q[i]);
        acc[2 * i + 1] += bf16hi_to_f32(q[i]);
      }
    }
  } else {
    for (long r = r0 + g; r < r1; r += kSumRows)
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (n + i < N) acc[i] += to_f32(x[r * N + n + i]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) part[g][8 * c + i] = acc[i];
  __syncthreads();
  const int t = threadIdx.x, col = blockIdx.x * kSumCols + t;
  if (t >= kSumCols || col >= N) return;
  float v = 0.0f;
#pragma unroll
  for (int i = 0; i < kSumRows; ++i) v += part[i][t];
  out[static_cast<long>(blockIdx.y) * N + col] = from_f32<TO>(v);
}
// rows of a chunk: 64 chunks at most, which the second pass reads in two steps, and
// enough for the card
int colsum_chunk(long M, int N) {
  const long across = (N + kSumCols - 1L) / kSumCols, want = std::min(64L, std::max(1L, 4096 / across));
  return static_cast<int>(std::max((M + want - 1) / want, 4L * kSumRows));
}

// tiles of BN columns, all matrices after each other
void cut_tiles(Fp8Segs& sg, int BN) {
  sg.blk0[0] = 0;
  for (int i = 0; i < kFp8Segs; ++i) sg.blk0[i + 1] = sg.blk0[i] + (i < sg.nseg ? (sg.N[i] + BN - 1) / BN : 0);
}
template <int CT, int R, int NW, int X>
void fp8_few(const Fp8X& in, Fp8Segs& sg, int M, int kb, hipStream_t s) {
  cut_tiles(sg, 16 * R);
  if (M > 16 * CT) sg.stream = 0;   // (rows of tiles share them)
  ProfScope prof_("fp8_few", s);
  hipLaunchKernelGGL((fp8_few_kernel<CT, R, NW, X>), dim3(sg.blk0[kFp8Segs] * ((M + 16 * CT - 1) / (16 * CT))),
                     dim3(64 * NW), 0, s, in, sg, M, kb);
}
template <int SN, int SM>
void fp8_large(const void* x, const void* xs, Fp8Segs& sg, int M, int kb, hipStream_t s) {
  cut_tiles(sg, 64 * SN);
  const int mtiles = (M + 64 * SM - 1) / (64 * SM);
  ProfScope prof_("fp8_large", s);
  hipLaunchKernelGGL((fp8_large_kernel<SN, SM>), dim3(sg.blk0[kFp8Segs] * mtiles), dim3(256), 0, s,
                     static_cast<const uint8_t*>(x), static_cast<const uint8_t*>(xs), sg, M, kb, mtiles);
}
template <int SN, int SM, int R, int OCC, int KS = 1, bool NT = false>
void fp8_ring(const void* x, const void* xs, Fp8Segs& sg, int M, int kb, hipStream_t s) {
  cut_tiles(sg, 64 * SN);
  const int mtiles = (M + 64 * SM - 1) / (64 * SM);
  ProfScope prof_("fp8_ring", s);
  hipLaunchKernelGGL((fp8_ring_kernel<SN, SM, R, OCC, KS, NT>), dim3(sg.blk0[kFp8Segs] * mtiles), dim3(256 * KS), 0, s,
                     static_cast<const uint8_t*>(x), static_cast<const uint8_t*>(xs), sg, M, kb, mtiles);
}

// The kernel by the sizes: the least estimate in us, of kb blocks of K, of
//   tiles <= 256      first(kb), one tile on each CU
//   more              again + (tiles / 256, between itself and its ceiling) each(kb)
// fitted to 131 products of 1 to 32768 rows, K 512 to 11008, N 1024 to 32000; the choice
// was at most 6 % behind the best of all, 0.5 % on average (linear8 in us, tiles of
// fp8_few, fp8_ring and fp8_large as rows x columns):
//   1 row, 1024 -> 1024       16 x 16 3.5   16 x 64 3.7    64 x 64 5.1
//   64 rows, 4096 -> 4096     16 x 16 15.5  16 x 64 8.2    64 x 64 11.0
//   200 rows, 8192 -> 1024    16 x 16 25.5  16 x 64 12.8   64 x 64 18.4
//   32 rows, 4096 -> 32000    16 x 32 43.2  64 x 64 28.5   64 x 128 25.5
//   500 rows, 2050 -> 4383    32 x 64 35.7  64 x 64 14.6   128 x 128 13.7  256 x 256 30.4
//   4000 rows, 1024 -> 4384   64 x 64 35.7  128 x 128 25.2 128 x 256 28.2  256 x 256 35.3
//   8192 rows, 4096 -> 4096   128 x 128 138 128 x 256 112  256 x 256 105
struct Fp8Shape {
  int bm, bn;
  float first0, first1, again, each0, each1;
};
constexpr int kFp8Few = 4;   // shapes of fp8_few, then tiles
constexpr Fp8Shape kFp8Shapes[] = {
    {16, 16, 3.5f, 0.0577f, 1.65f, 0.549f, 0.0717f},
    {16, 32, 3.52f, 0.0773f, 3.0f, 0.088f, 0.111f},
    {16, 64, 3.39f, 0.138f, 0.69f, 3.0f, 0.0957f},
    {32, 64, 3.83f, 0.219f, 1.6f, 1.9f, 0.2f},
    {64, 64, 3.2f, 0.235f, 3.55f, -0.17f, 0.258f},
    {64, 128, 4.0f, 0.321f, 3.84f, 0.109f, 0.38f},
    {128, 128, 4.64f, 0.461f, 4.0f, 0.26f, 0.574f},
    {128, 256, 7.76f, 0.745f, 5.17f, 1.94f, 0.865f},
    {256, 256, 8.2f, 1.1f, 2.2f, 7.8f, 1.43f},   // (full of such tiles the card is bound by power)
};
int fp8_shape(const Fp8Segs& sg, int M, int kb, float* per_cu) {
  constexpr int kShapes = sizeof(kFp8Shapes) / sizeof(kFp8Shapes[0]);
  int best = 0;
  float least = 0.0f;
  for (int i = 0; i < kShapes; ++i) {
    const Fp8Shape& p = kFp8Shapes[i];
    long tiles = 0;
    for (int k = 0; k < sg.nseg; ++k) tiles += (sg.N[k] + p.bn - 1) / p.bn;
    tiles *= (M + p.bm - 1) / p.bm;
    if (tiles >= 1 << 23) continue;   // (2^32 threads a grid, of up to 512 a tile)
    // (their line holds for one tile a CU alone: with more, 64 rows, 1024 -> 4384 would take
    // 16 x 64, 8.0 us, for 64 x 64, 5.4, and 400 rows, 4096 -> 1024 14.5 for 11.2)
    if ((i == 2 || i == 3) && tiles > 256) continue;
    const float r = static_cast<float>(tiles) / 256.0f, k = static_cast<float>(kb), each = p.each0 + p.each1 * k;
    float us = p.first0 + p.first1 * k;
    if (i < kFp8Few) us = std::max(us, p.again + r * each);
    else if (r > 1.0f) us = p.again + 0.5f * (r + static_cast<float>((tiles + 255) / 256)) * each;
    else if (i == kShapes - 1) us = std::max(us, r * (each + 2.0f));   // (300 rows, 1024 -> 32000: 20.8, for 19.0)
    if (least == 0.0f || us < least) {
      least = us;
      best = i;
      *per_cu = r;
    }
  }
  return best;
}

// Weights that one row of tiles reads and that take more than a third of the caches' 256
// MB pass them by: a model with one such weight has more weights than they hold.  From
// memory 1 row 4096 -> 32000 takes 26.5 us, so 23.8, 32 rows 27.6, so 24.2, 16 rows 4096 ->
// 24000 22.0, so 20.4; one weight alone, call after call, comes from the caches, 22.7, so
// 22.3, 21.6, so 22.8, and 16.8, so 18.2.  Smaller ones lose more there than they gain (64
// rows, 5120 -> 15000: 25 and 24, 16.3 and 22).
void fp8_stream(Fp8Segs& sg, int kb) {
  long bytes = 0;
  for (int i = 0; i < sg.nseg; ++i) bytes += (sg.N[i] + 15L) / 16 * kb * 2048;
  sg.stream = 3 * bytes > 256L << 20;
}

void fp8_go(const void* x, const void* xs, Fp8Segs& sg, int M, int kb, hipStream_t s) {
  const Fp8X in{x, xs, 0, 0, 0};
  if (M <= 64) fp8_stream(sg, kb);
  // few tiles a CU get deep rings (the smallest eight waves), more of them room beside each other
  float per_cu = 0.0f;
  switch (fp8_shape(sg, M, kb, &per_cu)) {
    case 0: return fp8_few<1, 1, 8, kCodes>(in, sg, M, kb, s);
    case 1: return fp8_few<1, 2, 8, kCodes>(in, sg, M, kb, s);
    case 2: return fp8_few<1, 4, 8, kCodes>(in, sg, M, kb, s);
    case 3: return fp8_few<2, 4, 8, kCodes>(in, sg, M, kb, s);
    case 4:
      return per_cu <= 1.0f && kb >= 8 ? fp8_ring<1, 1, 4, 2, 2>(x, xs, sg, M, kb, s)
                                       : fp8_ring<1, 1, 3, 5>(x, xs, sg, M, kb, s);
    case 5:
      return sg.stream ? fp8_ring<2, 1, 6, 2, 1, true>(x, xs, sg, M, kb, s)
                                  : fp8_ring<2, 1, 6, 2>(x, xs, sg, M, kb, s);
    case 6: return per_cu <= 2.0f ? fp8_ring<2, 2, 4, 2>(x, xs, sg, M, kb, s) : fp8_ring<2, 2, 3, 3>(x, xs, sg, M, kb, s);
    case 7: return fp8_ring<4, 2, 3, 2>(x, xs, sg, M, kb, s);
    default: return fp8_large<4, 4>(x, xs, sg, M, kb, s);
  }
}

// up to 16 rows in bfloat16, which every workgroup rounds again: tiles of 32 columns where
// those of 16 are more than the CUs (16 gated rows, 1024 -> 4384 4.9 us, by 16 7.6, 8192 -> 8192
// 20.8 and 36.3; 1 row without gate between 6 % less and 8 % more, 4096 -> 32000 29.1 and 27.0),
// of 16 where they are not (4096 -> 4096 11.2, by 32 11.5, 1 row 1024 -> 1024 3.05 and 3.65)
template <int X>
void fp8_go_bf16(const Fp8X& in, Fp8Segs& sg, int M, int kb, hipStream_t s) {
  fp8_stream(sg, kb);
  long tiles = 0;
  for (int i = 0; i < sg.nseg; ++i) tiles += (sg.N[i] + 15) / 16;
  if (tiles <= 256) fp8_few<1, 1, 8, X>(in, sg, M, kb, s);
  else fp8_few<1, 2, 8, X>(in, sg, M, kb, s);
}

// the weights of a call, checked
int fp8_matrices(const char* who, Fp8Segs& sg, int64_t M, int nseg, const int64_t* matrices) {
  SA_CHECK_ARG(nseg >= 1 && nseg <= kFp8Segs && matrices, "%s: %d weight matrices, 1..%d allowed", who, nseg, kFp8Segs);
  sg.nseg = nseg;
  long tiles = 0;
  for (int i = 0; i < nseg; ++i) {
    const int64_t* m = matrices + 5 * i;   // packed, scales, bias, y, N
    SA_CHECK_ARG(m[0] && m[1] && m[3] && m[4] > 0 && m[4] <= (1L << 24), "%s: weight matrix %d: null pointer or N %ld",
                 who, i, static_cast<long>(m[4]));
    SA_CHECK_ARG((m[0] & 15) == 0 && (m[1] & 3) == 0 && ((m[2] | m[3]) & 1) == 0, "%s: weight matrix %d is not aligned",
                 who, i);
    tiles += (m[4] + 63) / 64;
    sg.W[i] = reinterpret_cast<const uint8_t*>(m[0]);
    sg.scale[i] = reinterpret_cast<const uint8_t*>(m[1]);
    sg.bias[i] = reinterpret_cast<const bf16*>(m[2]);
    sg.y[i] = reinterpret_cast<bf16*>(m[3]);
    sg.N[i] = static_cast<int>(m[4]);
  }
  SA_CHECK_ARG(tiles * ((M + 63) / 64) < (1L << 23), "%s: %ld rows and %ld columns are too many", who,
               static_cast<long>(M), 64 * tiles);   // (tiles of 64 by 64 and more always fit a grid)
  return 0;
}

}  // namespace
}  // namespace sa

extern "C" int sa_fp8_linear(const void* codes, const void* scales, int64_t M, int K, int nseg,
                             const int64_t* matrices, void* stream) {
  const char* who = "sa_fp8_linear";
  SA_CHECK_ARG(M >= 1 && M <= (1 << 24) && K > 0 && K <= (1 << 22), "%s: M %ld must be 1..2^24 and K %d 1..2^22", who,
               static_cast<long>(M), K);
  SA_CHECK_ARG(codes && scales, "%s: null pointer", who);
  SA_CHECK_ARG(((reinterpret_cast<uintptr_t>(codes) & 15) | (reinterpret_cast<uintptr_t>(scales) & 3)) == 0,
               "%s: codes or scales of x are not aligned", who);
  sa::Fp8Segs sg{};
  if (const int rc = sa::fp8_matrices(who, sg, M, nseg, matrices)) return rc;
  sa::fp8_go(codes, scales, sg, static_cast<int>(M), (K + 127) / 128, static_cast<hipStream_t>(stream));
  SA_CHECK_LAUNCH(who);
  return 0;
}

extern "C" int sa_fp8_linear_bf16(const void* x, const void* xscale, int M, int K, int64_t ldx, int64_t ldg, int nseg,
                                  const int64_t* matrices, void* stream) {
  const char* who = "sa_fp8_linear_bf16";
  SA_CHECK_ARG(M >= 1 && M <= 16 && K > 0 && K <= (1 << 22), "%s: M %d must be 1..16 and K %d 1..2^22", who, M, K);
  SA_CHECK_ARG(x, "%s: null pointer", who);
  const uintptr_t at = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(xscale);
  SA_CHECK_ARG((at & 1) == 0, "%s: x and xscale are not aligned to their type", who);
  SA_CHECK_ARG(M == 1 || (ldx >= K && (!xscale || ldg >= K)), "%s: row strides %ld, %ld below K %d", who,
               static_cast<long>(ldx), static_cast<long>(ldg), K);
  sa::Fp8Segs sg{};
  if (const int rc = sa::fp8_matrices(who, sg, M, nseg, matrices)) return rc;
  const sa::Fp8X in{x, xscale, ldx, ldg, K};
  hipStream_t s = static_cast<hipStream_t>(stream);
  xscale ? sa::fp8_go_bf16<sa::kGated>(in, sg, M, (K + 127) / 128, s)
         : sa::fp8_go_bf16<sa::kBf16>(in, sg, M, (K + 127) / 128, s);
  SA_CHECK_LAUNCH(who);
  return 0;
}

extern "C" int sa_fp8_dequant_bf16(const void* packed, const void* scales, int N, int K, void* out, void* stream) {
  const char* who = "sa_fp8_dequant_bf16";
  SA_CHECK_ARG(N > 0 && K > 0, "%s: bad sizes N=%d K=%d", who, N, K);
  SA_CHECK_ARG(packed && scales && out, "%s: null pointer", who);
  SA_CHECK_ARG((reinterpret_cast<uintptr_t>(packed) & 7) == 0, "%s: packed weights are not aligned", who);
  const long kb = (K + 127L) / 128, blocks = ((N + 15L) / 16) * kb;
  SA_CHECK_ARG(blocks < (1L << 25), "%s: weights too large", who);   // (2^32 threads a grid)
  hipStream_t s = static_cast<hipStream_t>(stream);
  sa::ProfScope prof_("fp8_dequant", s);
  hipLaunchKernelGGL(sa::fp8_dequant_kernel, dim3(blocks), dim3(128), 0, s, static_cast<const uint8_t*>(packed),
                     static_cast<const uint8_t*>(scales), static_cast<sa::bf16*>(out), N, K, static_cast<int>(kb));
  SA_CHECK_LAUNCH(who);
  return 0;
}

extern "C" size_t sa_colsum_bf16_workspace_size(int64_t M, int N) {
  if (M < 1 || N < 1) return 0;
  const long chunk = sa::colsum_chunk(M, N), chunks = (M + chunk - 1) / chunk;
  return chunks > 1 ? static_cast<size_t>(chunks) * N * sizeof(float) : 0;
}

extern "C" int sa_colsum_bf16(const void* x, int64_t M, int N, void* out, void* workspace, size_t workspace_size,
                              void* stream) {
  const char* who = "sa_colsum_bf16";
  SA_CHECK_ARG(M >= 1 && M < (1L << 31) && N >= 1 && N <= (1 << 24), "%s: bad sizes M=%ld N=%d", who,
               static_cast<long>(M), N);
  SA_CHECK_ARG(x && out, "%s: null pointer", who);
  SA_CHECK_ARG(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) & 1) == 0 &&
                   (reinterpret_cast<uintptr_t>(workspace) & 3) == 0,
               "%s: a tensor is not aligned to its type", who);
  const size_t need = sa_colsum_bf16_workspace_size(M, N);
  SA_CHECK_ARG(need == 0 || (workspace && workspace_size >= need), "%s: workspace of %zu bytes, %zu needed", who,
               workspace ? workspace_size : 0, need);
  const int chunk = sa::colsum_chunk(M, N);
  const int chunks = static_cast<int>((M + chunk - 1) / chunk), across = (N + sa::kSumCols - 1) / sa::kSumCols;
  hipStream_t s = static_cast<hipStream_t>(stream);
  sa::ProfScope prof_("colsum", s);
  const auto* in = static_cast<const sa::bf16*>(x);
  auto* o = static_cast<sa::bf16*>(out);
  auto* ws = static_cast<float*>(workspace);
  if (chunks == 1) {
    hipLaunchKernelGGL((sa::colsum_kernel<sa::bf16, sa::bf16>), dim3(across), dim3(256), 0, s, in, o, M, N, chunk);
  } else {
    hipLaunchKernelGGL((sa::colsum_kernel<sa::bf16, float>), dim3(across, chunks), dim3(256), 0, s, in, ws, M, N, chunk);
    hipLaunchKernelGGL((sa::colsum_kernel<float, sa::bf16>), dim3(across), dim3(256), 0, s, ws, o,
                       static_cast<long>(chunks), N, chunks);
  }
  SA_CHECK_LAUNCH(who);
  return 0;
}
