// Activations kept in 8 bits between the forward and the backward pass (sm_100a): a tensor's codes and scales and back, RMSNorm
// whose normalised row is kept, SwiGLU whose gate and up are kept, and the backward passes that read them.
//
// Rows are cut into groups of 128 columns (the last of a row may be shorter).  With a the largest magnitude of a group,
//   int8  scale = a / 127, code = nearest integer of x * (127 / a);
//   e4m3  scale = the smallest power of two with a / scale <= 448: codes with exponents of their own gain nothing from a finer
//         scale, and with a power of two the only rounding is the code's own.  At most 2^119, with which the largest code stays
//         finite: a value above 1.75 * 2^127 (a mask of the type's lowest value) is clipped to that and does not read back as
//         infinity.
// A group whose magnitudes are all below 2^-100 has scale 0; one with an infinity or a NaN has scale NaN and reads back as NaN.
// A value reads back as code * scale, in fp32.
//
// Eight bits are what the caller asks for; everything in between (sums of squares, dot products, sigmoids, sums over rows) is fp32,
// and results are rounded to bf16 once.
//
// Everything here is bound by memory, SwiGLU by the issue of instructions almost as much: a thread has 16 columns of a row, eight
// threads share a group, and what is computed stays in registers.  WIDE: rows are whole 32-byte pieces and start on one, a thread's
// columns are one access of 32 bytes (16 of codes); otherwise they are two of 16 bytes (8 of codes), the second of which may lie
// beyond the row.
#include <atomic>

#include <cuda_fp16.h>

#include "common.cuh"
#include "launch.cuh"
#include "ody_kernels.h"
#include "sm100.cuh"

namespace ody {
namespace act8 {

constexpr int GROUP = 128;
enum { E4M3 = 0, INT8 = 1 };

// ------------------------------------------------------------------------------------------- pieces of a row

// 16 columns of a row in bf16, two a word, and their codes, four a word
struct Piece {
  uint32_t w[8];
};
struct Codes {
  uint32_t w[4];
};

// `both`: the second half is inside the row
template <bool WIDE>
__device__ __forceinline__ void load(Piece& p, const bf16* at, bool both) {
  if (WIDE) {
    asm volatile("ld.global.L1::no_allocate.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(p.w[0]), "=r"(p.w[1]), "=r"(p.w[2]), "=r"(p.w[3]), "=r"(p.w[4]), "=r"(p.w[5]), "=r"(p.w[6]), "=r"(p.w[7])
                 : "l"(at) : "memory");
  } else {
    const uint4 z = make_uint4(0, 0, 0, 0), a = reinterpret_cast<const uint4*>(at)[0], b = both ? reinterpret_cast<const uint4*>(at)[1] : z;
    p.w[0] = a.x; p.w[1] = a.y; p.w[2] = a.z; p.w[3] = a.w;
    p.w[4] = b.x; p.w[5] = b.y; p.w[6] = b.z; p.w[7] = b.w;
  }
}
template <bool WIDE>
__device__ __forceinline__ void store(bf16* at, const Piece& p, bool both) {
  if (WIDE) {
    asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(p.w[0]), "r"(p.w[1]), "r"(p.w[2]), "r"(p.w[3]),
                 "r"(p.w[4]), "r"(p.w[5]), "r"(p.w[6]), "r"(p.w[7]), "l"(at) : "memory");
  } else {
    reinterpret_cast<uint4*>(at)[0] = make_uint4(p.w[0], p.w[1], p.w[2], p.w[3]);
    if (both) reinterpret_cast<uint4*>(at)[1] = make_uint4(p.w[4], p.w[5], p.w[6], p.w[7]);
  }
}
template <bool WIDE>
__device__ __forceinline__ void load(Codes& c, const uint8_t* at, bool both) {
  if (WIDE) {
    const uint4 v = *reinterpret_cast<const uint4*>(at);
    c.w[0] = v.x; c.w[1] = v.y; c.w[2] = v.z; c.w[3] = v.w;
  } else {
    const uint2 a = reinterpret_cast<const uint2*>(at)[0], b = both ? reinterpret_cast<const uint2*>(at)[1] : make_uint2(0, 0);
    c.w[0] = a.x; c.w[1] = a.y; c.w[2] = b.x; c.w[3] = b.y;
  }
}
template <bool WIDE>
__device__ __forceinline__ void store(uint8_t* at, const Codes& c, bool both) {
  if (WIDE) {
    *reinterpret_cast<uint4*>(at) = make_uint4(c.w[0], c.w[1], c.w[2], c.w[3]);
  } else {
    reinterpret_cast<uint2*>(at)[0] = make_uint2(c.w[0], c.w[1]);
    if (both) reinterpret_cast<uint2*>(at)[1] = make_uint2(c.w[2], c.w[3]);
  }
}

// weights, which every row reads again
__device__ __forceinline__ void load_weight(Piece& p, const bf16* at, bool both) {
  const uint4 z = make_uint4(0, 0, 0, 0), a = reinterpret_cast<const uint4*>(at)[0], b = both ? reinterpret_cast<const uint4*>(at)[1] : z;
  p.w[0] = a.x; p.w[1] = a.y; p.w[2] = a.z; p.w[3] = a.w;
  p.w[4] = b.x; p.w[5] = b.y; p.w[6] = b.z; p.w[7] = b.w;
}

// Two columns as a packed pair of fp32
__device__ __forceinline__ uint64_t pair_of(uint32_t w) { return pk2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ uint32_t word_of(uint64_t v) {
  float a, b;
  upk2(v, a, b);
  const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&t);
}

// ------------------------------------------------------------------------------------------- codes and scales

// Largest magnitude of the group that this thread's columns belong to, as fp32 bits: bf16 magnitudes compare like integers, NaN
// above infinity above everything else.
__device__ __forceinline__ uint32_t group_top(const Piece& p) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = __vmaxu2(m, p.w[i] & 0x7fff7fffu);
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
  return max(m << 16, m & 0xffff0000u);
}

// scale, and what a value is multiplied with to become a code (a finite number always: 0 where the codes say nothing); called by
// whole warps
template <int FMT>
__device__ __forceinline__ void scale_of(uint32_t top, float& scale, float& inverse) {
  if (FMT == E4M3) {
    // a = 1.m * 2^e with 1.m up to 1.75: 448 = 1.75 * 2^8, the scale is 2^(e - 8), else one more
    const uint32_t e = min(((top + 0x1fffffu) >> 23) - 8, 246u);
    scale = __uint_as_float(e << 23);
    inverse = __uint_as_float((254 - e) << 23);
  } else {
    // Of two neighbours one divides for the scale and the other for its inverse, which is rounded up: a value of half the group's
    // largest stands on the border of 63 and 64, the even code, and with an inverse below 127 / a it fell to 63 (14 of bf16's 128
    // mantissas).  The other quotients of bf16 numbers are off their border by 2^-16 of themselves at least, or 127 / a is exact.
    const float a = __uint_as_float(top);
    const bool odd = threadIdx.x & 1;
    float mine = __fdiv_rn(odd ? 127.f : a, odd ? a : 127.f);
    if (odd && __fmaf_rn(mine, a, -127.f) < 0.f) mine = __uint_as_float(__float_as_uint(mine) + 1);
    const float other = __shfl_xor_sync(0xffffffffu, mine, 1);
    scale = odd ? other : mine;
    inverse = odd ? mine : other;
  }
  if (top < (27u << 23) || top >= 0x7f800000u) {
    scale = top < (27u << 23) ? 0.f : __uint_as_float(0x7fc00000u);
    inverse = 0.f;
  }
}

template <int FMT>
__device__ __forceinline__ Codes encode(const Piece& p, float inverse) {
  Codes c;
  // int8: x + 1.5 * 2^23 rounds x to the nearest integer (ties to even) into the low bits
  const uint64_t inv = pk2(inverse, inverse), magic = pk2(12582912.f, 12582912.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t v0 = pair_of(p.w[2 * i]), v1 = pair_of(p.w[2 * i + 1]);
    float a, b, d, e;
    upk2(FMT == E4M3 ? mul2(v0, inv) : fma2(v0, inv, magic), a, b);
    upk2(FMT == E4M3 ? mul2(v1, inv) : fma2(v1, inv, magic), d, e);
    if (FMT == E4M3) {
      uint16_t lo, hi;
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
      asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(e), "f"(d));
      c.w[i] = (uint32_t)lo | ((uint32_t)hi << 16);
    } else {
      const uint32_t lo = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040);
      const uint32_t hi = __byte_perm(__float_as_uint(d), __float_as_uint(e), 0x0040);
      c.w[i] = __byte_perm(lo, hi, 0x5410);
    }
  }
  return c;
}

// a word of codes as two pairs of fp32, not yet scaled.  Integers become fp32 in the conversion unit (CONVERT), which shares its
// rate with exponentials and quotients, or by arithmetic: code + 128 in the low byte of the half-precision 1024, less 1152.
// Neither alone keeps up with memory: 65536 x 4096 in int8 are restored in 125 us by conversions, 140 by arithmetic, 119 by both
// in turn; SwiGLU, which has exponentials, in 136 and 105.
template <int FMT, bool CONVERT>
__device__ __forceinline__ void decode4(uint32_t w, uint64_t& lo, uint64_t& hi) {
  if (FMT == INT8 && CONVERT) {
    lo = pk2((float)(int8_t)w, (float)(int8_t)(w >> 8));
    hi = pk2((float)(int8_t)(w >> 16), (float)(int8_t)(w >> 24));
    return;
  }
  uint32_t h0, h1;
  if (FMT == E4M3) {
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h0) : "h"((uint16_t)(w & 0xffffu)));
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h1) : "h"((uint16_t)(w >> 16)));
  } else {
    const uint32_t u = w ^ 0x80808080u;
    h0 = __byte_perm(u, 0x64646464u, 0x4140);
    h1 = __byte_perm(u, 0x64646464u, 0x4342);
  }
  __half2 a = *reinterpret_cast<const __half2*>(&h0), b = *reinterpret_cast<const __half2*>(&h1);
  if (FMT == INT8) {
    const __half2 off = __floats2half2_rn(-1152.f, -1152.f);
    a = __hadd2(a, off);
    b = __hadd2(b, off);
  }
  const float2 fa = __half22float2(a), fb = __half22float2(b);
  lo = pk2(fa.x, fa.y);
  hi = pk2(fb.x, fb.y);
}

// ------------------------------------------------------------------------------------------- rows over threads

// A block covers `tile_groups` groups of `rows` rows at a time; a row's threads are eight a group, so that a group lies in one warp.
struct Split {
  int row_threads, rows, tiles, tile_groups, groups, threads;
};
static Split split_of(int n) {
  Split s;
  s.groups = (n + GROUP - 1) / GROUP;
  s.tiles = (s.groups * 8 + 255) / 256;
  s.tile_groups = (s.groups + s.tiles - 1) / s.tiles;
  s.row_threads = s.tile_groups * 8;
  s.rows = 256 / s.row_threads;
  s.threads = (s.rows * s.row_threads + 31) / 32 * 32;
  return s;
}

// This thread's place: first row (the others follow every `rows` rows), column, and whether it has any
struct Place {
  int64_t row, block;                                          // the thread's, the block's
  int col, group;
  bool on, both, first;                                        // first: the thread that writes the group's scale
};
__device__ __forceinline__ Place place_of(const Split& s, int n, int U) {
  const int tile = blockIdx.x % s.tiles, block = blockIdx.x / s.tiles;
  const int r = threadIdx.x / s.row_threads, t = threadIdx.x - r * s.row_threads;
  Place p;
  p.block = (int64_t)block * (s.rows * U);
  p.row = p.block + r;
  p.col = tile * s.tile_groups * GROUP + t * 16;
  p.group = p.col / GROUP;
  p.on = r < s.rows && p.col < n;
  p.both = p.col + 8 < n;
  p.first = p.on && t % 8 == 0;
  return p;
}
static unsigned blocks_of(const Split& s, int64_t rows, int u) {
  const int64_t per = (int64_t)s.rows * u;
  return (unsigned)((rows + per - 1) / per * s.tiles);
}

// How many rows after one another a block has: one below sixteen blocks an SM, above as many as leave eight, up to four, so that what
// it takes to start is little of its time (index arithmetic of a hundred instructions, as many as half a row's)
static int rows_a_block(const Split& s, int64_t rows) {
  const int64_t blocks = (rows + s.rows - 1) / s.rows * s.tiles, per = blocks / (148 * 8);
  return (int)(per < 1 ? 1 : per > 4 ? 4 : per);
}

// ------------------------------------------------------------------------------------------- a tensor and back

// U rows of a thread under way at once, and as many blocks as that takes.  65536 x 4096: 118 us in e4m3 and 115 in int8, 6.9 TB/s
// of what is read and written; 65536 x 4104, in two accesses of 16 bytes, 120 and 130.
template <int FMT, bool WIDE, int U>
__global__ void __launch_bounds__(256) pack8_k(const bf16* x, int64_t ldx, uint8_t* __restrict__ codes, float* __restrict__ scales,
                                               int64_t rows, int n, Split s) {
  after_previous_kernel(x);
  const Place at = place_of(s, n, U);
  Piece p[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t row = at.row + (int64_t)u * s.rows;
    p[u] = Piece{};
    if (at.on && row < rows) load<WIDE>(p[u], x + row * ldx + at.col, at.both);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t row = at.row + (int64_t)u * s.rows;
    float scale, inverse;
    scale_of<FMT>(group_top(p[u]), scale, inverse);
    if (at.on && row < rows) {
      store<WIDE>(codes + row * n + at.col, encode<FMT>(p[u], inverse), at.both);
      if (at.first) scales[row * s.groups + at.group] = scale;
    }
  }
}

// w (bf16, may be null): each column times its weight.  65536 x 4096: 119 us in either format, 6.8 TB/s.
template <int FMT, bool WIDE, int U>
__global__ void __launch_bounds__(256) unpack8_k(const uint8_t* codes, const float* scales, const bf16* w, bf16* __restrict__ x,
                                                 int64_t rows, int n, Split s) {
  after_previous_kernel(codes, scales, w);
  const Place at = place_of(s, n, U);
  if (!at.on) return;
  Codes c[U];
  float scale[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t row = at.row + (int64_t)u * s.rows;
    if (row < rows) {
      load<WIDE>(c[u], codes + row * n + at.col, at.both);
      scale[u] = scales[row * s.groups + at.group];
    }
  }
  Piece wp;
  if (w != nullptr) load_weight(wp, w + at.col, at.both);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t row = at.row + (int64_t)u * s.rows;
    if (row >= rows) break;
    Piece o;
    const uint64_t sc = pk2(scale[u], scale[u]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint64_t lo, hi;
      if (i & 1) decode4<FMT, true>(c[u].w[i], lo, hi);
      else decode4<FMT, false>(c[u].w[i], lo, hi);
      lo = mul2(lo, sc);
      hi = mul2(hi, sc);
      if (w != nullptr) {
        lo = mul2(lo, pair_of(wp.w[2 * i]));
        hi = mul2(hi, pair_of(wp.w[2 * i + 1]));
      }
      o.w[2 * i] = word_of(lo);
      o.w[2 * i + 1] = word_of(hi);
    }
    store<WIDE>(x + row * n + at.col, o, at.both);
  }
}

// ------------------------------------------------------------------------------------------- SwiGLU

__device__ __forceinline__ float reciprocal(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// p = sigmoid(g) of two gates, and pp = p (1 - p).  With t = exp(-|g|), r = 1 / (1 + t) and q = t r: p is r or q, and pp = q r.
// Divisors are 1 to 2, and nothing overflows; a t below 2^-126 counts as zero.  The quick forms of both functions, for these kernels
// are bound by the issue of instructions almost as much as by memory: the exponent is rounded to fp32 before, so that t is off by
// up to |g| 2^-23 + 2^-21 of itself (2^-16.5 where t ends), and so are q and p of a negative g; r, and p of a positive one, by 2^-21.
__device__ __forceinline__ uint64_t sigmoid(uint64_t g, uint64_t& pp) {
  float a, b, ra, rb, qa, qb;
  upk2(mul2(g, pk2(1.4426950408889634f, 1.4426950408889634f)), a, b);
  const uint64_t t = pk2(exp2_mufu(-fabsf(a)), exp2_mufu(-fabsf(b)));
  upk2(add2(t, pk2(1.f, 1.f)), ra, rb);
  const uint64_t r = pk2(reciprocal(ra), reciprocal(rb)), q = mul2(t, r);
  pp = mul2(q, r);
  upk2(r, ra, rb);
  upk2(q, qa, qb);
  return pk2(a < 0.f ? qa : ra, b < 0.f ? qb : rb);
}
__device__ __forceinline__ uint64_t silu(uint64_t g) {
  uint64_t pp;
  return mul2(g, sigmoid(g, pp));
}

// h = silu(g) u from gu = [gate | up]; both halves are kept, each in groups from its own first column.  Four blocks an SM: with
// registers for one more it takes as long, for two more 218 us in place of 168 (32768 x 4096, e4m3).  32768 x 5504: 229 us in e4m3
// (6.4 TB/s), 239 in int8; with one row a block 245.
template <int FMT, bool WIDE>
__global__ void __launch_bounds__(256, 4) swiglu8_fwd_k(const bf16* gu, bf16* __restrict__ h, uint8_t* __restrict__ codes,
                                                        float* __restrict__ scales, int64_t rows, int n, Split s, int per) {
  after_previous_kernel(gu);
  const Place at = place_of(s, n, per);
#pragma unroll 1
  for (int k = 0; k < per; ++k) {
    const int64_t row = at.row + (int64_t)k * s.rows;
    if (at.block + (int64_t)k * s.rows >= rows) break;         // for the whole block: its warps exchange magnitudes
    const bool on = at.on && row < rows;
    Piece g{}, u{};
    if (on) {
      const bf16* src = gu + row * 2 * n + at.col;
      load<WIDE>(g, src, at.both);
      load<WIDE>(u, src + n, at.both);
    }
    float gs, gi, us, ui;
    scale_of<FMT>(group_top(g), gs, gi);
    scale_of<FMT>(group_top(u), us, ui);
    if (!on) continue;
    uint8_t* dst = codes + row * 2 * n + at.col;
    store<WIDE>(dst, encode<FMT>(g, gi), at.both);
    store<WIDE>(dst + n, encode<FMT>(u, ui), at.both);
    if (at.first) {
      float* sp = scales + row * 2 * s.groups + at.group;
      sp[0] = gs;
      sp[s.groups] = us;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) g.w[i] = word_of(mul2(silu(pair_of(g.w[i])), pair_of(u.w[i])));
    store<WIDE>(h + row * n + at.col, g, at.both);
  }
}

// h again, from what was kept; the next row's codes under way while a row is computed.  32768 x 5504: 133 us in e4m3 (5.5 TB/s), 138
// in int8, bound by about 200 instructions for 16 columns; with one row a block and nothing ahead 185.
template <int FMT, bool WIDE>
__global__ void __launch_bounds__(256, 5) swiglu8_restore_k(const uint8_t* codes, const float* scales, bf16* __restrict__ h, int64_t rows,
                                                            int n, Split s, int per) {
  after_previous_kernel(codes, scales);
  const Place at = place_of(s, n, per);
  if (!at.on) return;
  Codes cg, cu;
  float gs = 0.f, us = 0.f;
  auto fetch = [&](int64_t row) {
    const uint8_t* src = codes + row * 2 * n + at.col;
    load<WIDE>(cg, src, at.both);
    load<WIDE>(cu, src + n, at.both);
    const float* sp = scales + row * 2 * s.groups + at.group;
    gs = sp[0];
    us = sp[s.groups];
  };
  if (at.row < rows) fetch(at.row);
#pragma unroll 1
  for (int k = 0; k < per; ++k) {
    const int64_t row = at.row + (int64_t)k * s.rows;
    if (row >= rows) break;
    const Codes g4 = cg, u4 = cu;
    const uint64_t sg = pk2(gs, gs), su = pk2(us, us);
    if (k + 1 < per && row + s.rows < rows) fetch(row + s.rows);      // under way while this row is computed
    Piece o;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint64_t g[2], u[2];
      decode4<FMT, false>(g4.w[i], g[0], g[1]);
      decode4<FMT, false>(u4.w[i], u[0], u[1]);
#pragma unroll
      for (int j = 0; j < 2; ++j) o.w[2 * i + j] = word_of(mul2(silu(mul2(g[j], sg)), mul2(u[j], su)));
    }
    store<WIDE>(h + row * n + at.col, o, at.both);
  }
}

// With p = sigmoid(g): dg = dh u (p + g p (1 - p)), du = dh g p, from what was kept.  One row a block (four: 159 -> 177 us at 32768 x
// 4096).  32768 x 5504: 214 us in e4m3 (6.8 TB/s), 218 in int8.
template <int FMT, bool WIDE>
__global__ void __launch_bounds__(256, 6) swiglu8_bwd_k(const bf16* dh, const uint8_t* codes, const float* scales, bf16* __restrict__ dgu,
                                                        int64_t rows, int n, Split s) {
  after_previous_kernel(dh, codes, scales);
  const Place at = place_of(s, n, 1);
  if (!at.on || at.row >= rows) return;
  Piece d, og;
  Codes cg, cu;
  load<WIDE>(d, dh + at.row * n + at.col, at.both);
  const uint8_t* src = codes + at.row * 2 * n + at.col;
  load<WIDE>(cg, src, at.both);
  load<WIDE>(cu, src + n, at.both);
  const float* sp = scales + at.row * 2 * s.groups + at.group;
  const uint64_t sg = pk2(sp[0], sp[0]), su = pk2(sp[s.groups], sp[s.groups]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint64_t g[2], u[2];
    decode4<FMT, false>(cg.w[i], g[0], g[1]);
    decode4<FMT, false>(cu.w[i], u[0], u[1]);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const uint64_t gv = mul2(g[j], sg), uv = mul2(u[j], su), dv = pair_of(d.w[2 * i + j]);
      uint64_t pp;
      const uint64_t p = sigmoid(gv, pp);
      d.w[2 * i + j] = word_of(mul2(dv, mul2(gv, p)));
      og.w[2 * i + j] = word_of(mul2(mul2(dv, uv), fma2(gv, pp, p)));
    }
  }
  bf16* dst = dgu + at.row * 2 * n + at.col;
  store<WIDE>(dst, og, at.both);
  store<WIDE>(dst + n, d, at.both);
}

// ------------------------------------------------------------------------------------------- RMSNorm

// s = x (+ delta, rounded as the stream is stored), r = rsqrt(mean s^2 + eps), y = s r w.  What is kept is the row without the
// weight, s r: the codes of s, and its scales times r.  The row stays in registers, NP pieces a thread, of one warp (ONE, up to 1024
// columns: eight rows a block, no barrier) or of a block that is as wide as the row wants.  What bounds it is how much of the next
// rows is under way while a block waits for its sum.  With the addition a thread has two pieces to load, and what counts is blocks
// an SM: 40 registers, for which the weights are read late.  Without it a block has R = 2 rows, and reads the weights early.
// 65536 x 4096: 204 us (6.6 TB/s; one row a block 223), with the addition 352 (6.9 TB/s); 32768 x 8192: 220 (308) and 350 (385).
template <int FMT, bool WIDE, bool DELTA, bool ONE, int NP, int R>
__global__ void __launch_bounds__(ONE ? 256 : 512, ONE ? 1 : DELTA && NP == 1 ? 3 : 2)
    rmsnorm8_fwd_k(const bf16* x, const bf16* delta, const bf16* w, bf16* __restrict__ sum_out, bf16* __restrict__ y,
                   float* __restrict__ rstd, uint8_t* __restrict__ codes, float* __restrict__ scales, int64_t rows, int n, float eps) {
  after_previous_kernel(x, delta, w);
  const int warp = threadIdx.x >> 5, threads = ONE ? 32 : blockDim.x;
  const int64_t row = (ONE ? (int64_t)blockIdx.x * 8 + warp : (int64_t)blockIdx.x) * R;
  if (row >= rows) return;                                     // a whole warp (ONE)
  const int t = ONE ? threadIdx.x & 31 : threadIdx.x;
  const int here = R == 1 || rows - row >= R ? R : (int)(rows - row);
  const int64_t base = row * n;
  Piece p[R][NP];
#pragma unroll
  for (int k = 0; k < R; ++k)
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = (t + i * threads) * 16;
      p[k][i] = Piece{};
      if (c < n && k < here) load<WIDE>(p[k][i], x + base + (int64_t)k * n + c, c + 8 < n);
    }
  if (DELTA) {
    Piece d[R][NP];
#pragma unroll
    for (int k = 0; k < R; ++k)
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int c = (t + i * threads) * 16;
        d[k][i] = Piece{};
        if (c < n && k < here) load<WIDE>(d[k][i], delta + base + (int64_t)k * n + c, c + 8 < n);
      }
#pragma unroll
    for (int k = 0; k < R; ++k)
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int c = (t + i * threads) * 16;
#pragma unroll
        for (int j = 0; j < 8; ++j) p[k][i].w[j] = word_of(add2(pair_of(p[k][i].w[j]), pair_of(d[k][i].w[j])));
        if (c < n && k < here) store<WIDE>(sum_out + base + (int64_t)k * n + c, p[k][i], c + 8 < n);
      }
  }
  constexpr bool EARLY = !DELTA && !ONE;                                // weights under way while the rows are summed
  Piece wp[NP];
  if (EARLY)
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = (t + i * threads) * 16;
      if (c < n) load_weight(wp[i], w + c, c + 8 < n);
    }
  float ss[R];
#pragma unroll
  for (int k = 0; k < R; ++k) {
    uint64_t ss2 = pk2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint64_t v = pair_of(p[k][i].w[j]);
        ss2 = fma2(v, v, ss2);
      }
    float a, b;
    upk2(ss2, a, b);
    ss[k] = warp_sum(a + b);
  }
  if (!ONE) {
    __shared__ float red[R][16];
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int k = 0; k < R; ++k) red[k][warp] = ss[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < R; ++k) {
      ss[k] = 0.f;
      for (int i = 0; i < threads >> 5; ++i) ss[k] += red[k][i];
    }
  }
  const int groups = (n + GROUP - 1) / GROUP;
#pragma unroll
  for (int k = 0; k < R; ++k) {
    const float r = rsqrtf(ss[k] / (float)n + eps);
    if (t == 0 && k < here) rstd[row + k] = r;
    const uint64_t rr = pk2(r, r);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = (t + i * threads) * 16;
      const int64_t at = base + (int64_t)k * n + c;
      float scale, inverse;
      scale_of<FMT>(group_top(p[k][i]), scale, inverse);
      if (c < n && k < here) {
        store<WIDE>(codes + at, encode<FMT>(p[k][i], inverse), c + 8 < n);
        if (c % GROUP == 0) scales[(row + k) * groups + c / GROUP] = scale * r;
        if (!EARLY) load_weight(wp[i], w + c, c + 8 < n);
#pragma unroll
        for (int j = 0; j < 8; ++j) p[k][i].w[j] = word_of(mul2(mul2(pair_of(p[k][i].w[j]), rr), pair_of(wp[i].w[j])));
        store<WIDE>(y + at, p[k][i], c + 8 < n);
      }
    }
  }
}

// With g = dy w, x' the kept row and r its 1 / rms: dx = r (g - x' mean(g x')) (+ ds), and dw the sum over the rows of dy x'.
// A block keeps the sums of its columns in registers over all its rows; ody_colsum adds the blocks up.  Rows of dy, ds, codes and
// scales come through a ring of asynchronous copies: a thread copies exactly what it reads itself, so that the ring needs no
// barrier, and the next rows are under way while a row's dot product waits at its own.  65536 x 4096 with ds: 275 us (6.9 TB/s); 2048 x
// 4096: 17, of which the ring's first rows and the sum over the blocks are half.
template <int N>
__device__ __forceinline__ void copy_async(void* dst, const void* src) {
  if (N == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "n"(N) : "memory");
}

// A stage of the ring: NP pieces of 8 columns a thread, each array with an entry a thread
template <int NP>
struct Stage {
  uint4 *dy, *ds;
  uint2* codes;
  float* scale;
  __device__ __forceinline__ Stage(uint8_t* ring, int stage) {
    const int t = blockDim.x;
    uint8_t* p = ring + stage * NP * t * BYTES + threadIdx.x * 16;
    dy = reinterpret_cast<uint4*>(p);
    ds = reinterpret_cast<uint4*>(p + NP * t * 16);
    codes = reinterpret_cast<uint2*>(ring + stage * NP * t * BYTES + NP * t * 32 + threadIdx.x * 8);
    scale = reinterpret_cast<float*>(ring + stage * NP * t * BYTES + NP * t * 40 + threadIdx.x * 4);
  }
  static constexpr int BYTES = 44;                             // a piece
};

template <int FMT, int NP, int STAGES, int THREADS, int BLOCKS>
__global__ void __launch_bounds__(THREADS, BLOCKS) rmsnorm8_bwd_k(const bf16* dy, const uint8_t* codes, const float* scales,
                                                          const bf16* w, const float* rstd, const bf16* ds, bf16* __restrict__ dx,
                                                          float* __restrict__ dw_partial, int64_t rows, int n) {
  after_previous_kernel(dy, codes, scales, w, rstd, ds);
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ __align__(16) float red[2][16];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5, T = blockDim.x;
  const int groups = (n + GROUP - 1) / GROUP;
  uint64_t acc[NP][4];
  uint4 wv[NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int c = (tid + i * T) * 8;
    wv[i] = c < n ? *reinterpret_cast<const uint4*>(w + c) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = pk2(0.f, 0.f);
  }
  if (tid < 32) red[tid >> 4][tid & 15] = 0.f;                 // warps that there are none of
  __syncthreads();
  auto fetch = [&](int64_t row, int stage) {
    if (row < rows) {
      const Stage<NP> to(ring, stage);
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const int c = (tid + i * T) * 8;
        if (c < n) {
          copy_async<16>(to.dy + i * T, dy + row * n + c);
          if (ds != nullptr) copy_async<16>(to.ds + i * T, ds + row * n + c);
          copy_async<8>(to.codes + i * T, codes + row * n + c);
          copy_async<4>(to.scale + i * T, scales + row * groups + c / GROUP);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // dy, g = dy w and x' of one piece of the row in a stage
  auto piece = [&](const Stage<NP>& from, int i, uint64_t* d, uint64_t* g, uint64_t* xh) {
    const uint4 d4 = from.dy[i * T];
    const uint2 c2 = from.codes[i * T];
    const float sc = from.scale[i * T];
    const uint32_t dw[4] = {d4.x, d4.y, d4.z, d4.w}, ww[4] = {wv[i].x, wv[i].y, wv[i].z, wv[i].w};
    decode4<FMT, true>(c2.x, xh[0], xh[1]);
    decode4<FMT, false>(c2.y, xh[2], xh[3]);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      xh[j] = mul2(xh[j], pk2(sc, sc));
      d[j] = pair_of(dw[j]);
      g[j] = mul2(d[j], pair_of(ww[j]));
    }
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) fetch(blockIdx.x + (int64_t)s * gridDim.x, s);
  const float inv_n = 1.f / (float)n;
  int par = 0, stage = 0;
  float r = (int64_t)blockIdx.x < rows ? rstd[blockIdx.x] : 0.f;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, par ^= 1) {
    const int64_t next = row + gridDim.x;
    const float r_next = next < rows ? rstd[next] : 0.f;
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    constexpr bool KEEP = NP <= 2;                             // wider rows are read from the ring again: registers
    const Stage<NP> from(ring, stage);
    uint64_t g[KEEP ? NP : 1][4], xh[KEEP ? NP : 1][4];
    uint64_t dot2 = pk2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = (tid + i * T) * 8, k = KEEP ? i : 0;
      if (c < n) {
        uint64_t d[4];
        piece(from, i, d, g[k], xh[k]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[i][j] = fma2(d[j], xh[k][j], acc[i][j]);
          dot2 = fma2(g[k][j], xh[k][j], dot2);
        }
      }
    }
    // into the slot of the row before this one, which this thread is done with
    fetch(row + (int64_t)(STAGES - 1) * gridDim.x, stage == 0 ? STAGES - 1 : stage - 1);
    float a, b;
    upk2(dot2, a, b);
    float dot = warp_sum(a + b);
    if (lane == 0) red[par][wid] = dot;
    __syncthreads();
    dot = 0.f;
#pragma unroll
    for (int i = 0; i < THREADS / 128; ++i) {
      const float4 v = *reinterpret_cast<const float4*>(&red[par][4 * i]);
      dot += (v.x + v.y) + (v.z + v.w);
    }
    dot *= inv_n;
    const uint64_t minus = pk2(-dot, -dot), rr = pk2(r, r);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int c = (tid + i * T) * 8, k = KEEP ? i : 0;
      if (c < n) {
        if (!KEEP) {
          uint64_t d[4];
          piece(from, i, d, g[k], xh[k]);
        }
        uint4 add = make_uint4(0, 0, 0, 0);
        if (ds != nullptr) add = from.ds[i * T];
        const uint32_t a4[4] = {add.x, add.y, add.z, add.w};
        uint32_t o[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint64_t v = fma2(xh[k][j], minus, g[k][j]);
          o[j] = word_of(ds != nullptr ? fma2(v, rr, pair_of(a4[j])) : mul2(v, rr));
        }
        *reinterpret_cast<uint4*>(dx + row * n + c) = make_uint4(o[0], o[1], o[2], o[3]);
      }
    }
    r = r_next;
    if (++stage == STAGES) stage = 0;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int c = (tid + i * T) * 8;
    if (c < n) {
      uint64_t* p = reinterpret_cast<uint64_t*>(dw_partial + (int64_t)blockIdx.x * n + c);
#pragma unroll
      for (int j = 0; j < 4; ++j) p[j] = acc[i][j];
    }
  }
}

}  // namespace act8
}  // namespace ody

// =========================================================================================== launchers

using namespace ody;
using namespace ody::act8;

static int last_err() { return (int)cudaGetLastError(); }
static bool aligned(const void* p, uintptr_t to) { return p == nullptr || ((uintptr_t)p & (to - 1)) == 0; }
static bool bad_rows(int64_t rows, int n, int fmt) { return rows < 0 || n <= 0 || n % 8 != 0 || (fmt != E4M3 && fmt != INT8); }

// A launch for each format and width of a piece
#define FMT_WIDE(kernel, ...)                                                                             \
  do {                                                                                                 \
    if (fmt == E4M3) { if (wide) kernel(E4M3, true, __VA_ARGS__); else kernel(E4M3, false, __VA_ARGS__); } \
    else { if (wide) kernel(INT8, true, __VA_ARGS__); else kernel(INT8, false, __VA_ARGS__); }             \
  } while (0)

extern "C" int ody_pack8(const void* x, int64_t ldx, void* codes, float* scales, int64_t rows, int n, int fmt, cudaStream_t st) {
  if (bad_rows(rows, n, fmt) || ldx % 8 != 0 || !aligned(x, 16) || !aligned(codes, 8)) return (int)cudaErrorInvalidValue;
  if (rows == 0) return 0;
  const bool wide = n % 16 == 0 && ldx % 16 == 0 && aligned(x, 32) && aligned(codes, 16);
  const Split s = split_of(n);
#define L(F, W, U) launch_kernel(pack8_k<F, W, U>, blocks_of(s, rows, U), s.threads, 0, st, 1, (const bf16*)x, ldx, (uint8_t*)codes, scales, rows, n, s)
  FMT_WIDE(L, 2);
#undef L
  return last_err();
}

extern "C" int ody_unpack8(const void* codes, const float* scales, const void* w, void* x, int64_t rows, int n, int fmt, cudaStream_t st) {
  if (bad_rows(rows, n, fmt) || !aligned(x, 16) || !aligned(w, 16) || !aligned(codes, 8)) return (int)cudaErrorInvalidValue;
  if (rows == 0) return 0;
  const bool wide = n % 16 == 0 && aligned(x, 32) && aligned(w, 32) && aligned(codes, 16);
  const Split s = split_of(n);
#define L(F, W, U) launch_kernel(unpack8_k<F, W, U>, blocks_of(s, rows, U), s.threads, 0, st, 1, (const uint8_t*)codes, scales, (const bf16*)w, (bf16*)x, rows, n, s)
  FMT_WIDE(L, 2);
#undef L
  return last_err();
}

extern "C" int ody_swiglu8_fwd(const void* gu, void* h, void* codes, float* scales, int64_t rows, int n, int fmt, cudaStream_t st) {
  if (bad_rows(rows, n, fmt) || !aligned(gu, 16) || !aligned(h, 16) || !aligned(codes, 8)) return (int)cudaErrorInvalidValue;
  if (rows == 0) return 0;
  const bool wide = n % 16 == 0 && aligned(gu, 32) && aligned(h, 32) && aligned(codes, 16);
  const Split s = split_of(n);
  const int per = rows_a_block(s, rows);
#define L(F, W, U) launch_kernel(swiglu8_fwd_k<F, W>, blocks_of(s, rows, U), s.threads, 0, st, 1, (const bf16*)gu, (bf16*)h, (uint8_t*)codes, scales, rows, n, s, U)
  FMT_WIDE(L, per);
#undef L
  return last_err();
}

extern "C" int ody_swiglu8_restore(const void* codes, const float* scales, void* h, int64_t rows, int n, int fmt, cudaStream_t st) {
  if (bad_rows(rows, n, fmt) || !aligned(h, 16) || !aligned(codes, 8)) return (int)cudaErrorInvalidValue;
  if (rows == 0) return 0;
  const bool wide = n % 16 == 0 && aligned(h, 32) && aligned(codes, 16);
  const Split s = split_of(n);
  const int per = rows_a_block(s, rows);
#define L(F, W, U) launch_kernel(swiglu8_restore_k<F, W>, blocks_of(s, rows, U), s.threads, 0, st, 1, (const uint8_t*)codes, scales, (bf16*)h, rows, n, s, U)
  FMT_WIDE(L, per);
#undef L
  return last_err();
}

extern "C" int ody_swiglu8_bwd(const void* dh, const void* codes, const float* scales, void* dgu, int64_t rows, int n, int fmt,
                               cudaStream_t st) {
  if (bad_rows(rows, n, fmt) || !aligned(dh, 16) || !aligned(dgu, 16) || !aligned(codes, 8)) return (int)cudaErrorInvalidValue;
  if (rows == 0) return 0;
  const bool wide = n % 16 == 0 && aligned(dh, 32) && aligned(dgu, 32) && aligned(codes, 16);
  const Split s = split_of(n);
#define L(F, W, U) launch_kernel(swiglu8_bwd_k<F, W>, blocks_of(s, rows, U), s.threads, 0, st, 1, (const bf16*)dh, (const uint8_t*)codes, scales, (bf16*)dgu, rows, n, s)
  FMT_WIDE(L, 1);
#undef L
  return last_err();
}

extern "C" int ody_rmsnorm8_fwd(const void* x, const void* delta, const void* w, void* sum_out, void* y, float* rstd, void* codes,
                                float* scales, int64_t rows, int n, float eps, int fmt, cudaStream_t st) {
  if (bad_rows(rows, n, fmt) || n > ODY_RMSNORM8_MAX || !aligned(x, 16) || !aligned(delta, 16) || !aligned(w, 16) || !aligned(sum_out, 16) ||
      !aligned(y, 16) || !aligned(codes, 8) || (delta != nullptr) != (sum_out != nullptr))
    return (int)cudaErrorInvalidValue;
  if (rows == 0) return 0;
  const bool wide = n % 16 == 0 && aligned(x, 32) && aligned(delta, 32) && aligned(w, 32) && aligned(sum_out, 32) && aligned(y, 32) && aligned(codes, 16);
  const int pieces = (n + 15) / 16;
#define L(F, W, D, ONE, P, R)                                                                                                         \
  launch_kernel(rmsnorm8_fwd_k<F, W, D, ONE, P, R>, (unsigned)((rows + (ONE ? 8 : 1) * R - 1) / ((ONE ? 8 : 1) * R)),                      \
                ONE ? 256 : (pieces + 32 * P - 1) / (32 * P) * 32, 0, st, 1, (const bf16*)x, (const bf16*)delta, (const bf16*)w,             \
                (bf16*)sum_out, (bf16*)y, rstd, (uint8_t*)codes, scales, rows, n, eps)
#define ROW(F, W, unused)                                                                                                             \
  do {                                                                                                                                \
    if (delta != nullptr) {                                                                                                           \
      if (pieces <= 32) L(F, W, true, true, 1, 1); else if (pieces <= 64) L(F, W, true, true, 2, 1);                                    \
      else if (pieces <= 512) L(F, W, true, false, 1, 1); else L(F, W, true, false, 2, 1);                                              \
    } else {                                                                                                                          \
      if (pieces <= 32) L(F, W, false, true, 1, 1); else if (pieces <= 64) L(F, W, false, true, 2, 1);                                    \
      else if (pieces <= 512) L(F, W, false, false, 1, 2); else L(F, W, false, false, 2, 1);                                              \
    }                                                                                                                                 \
  } while (0)
  FMT_WIDE(ROW, 0);
#undef ROW
#undef L
  return last_err();
}

// Pieces of 8 columns a thread has, threads of a block, and blocks: sixteen an SM at most, for the sum over the blocks reads a row of
// each, and of up to 600 threads together, which are eighteen warps; with 108 registers (94 with one piece) that many have room.
// Blocks as wide as their rows: of 65536 rows 256 wide the gradient takes 25 us, with blocks of 256 threads 92; of 32768 rows 8192
// wide 284 with two pieces a thread, 360 with four and half the threads.  Blocks of nine to sixteen warps are not as good throughout: of
// 32768 rows the gradient with ds runs at 1.02 of the copy rate with 4096 columns, 0.70 with 4104, 0.76 with 4608 and 4616, 0.84 with
// 5120, 0.94 with 6144, 0.96 with 7168 and 1.01 with 8192.  Wider rows have room for 256 threads with up to eight pieces: of
// 16384 rows 11008 wide 232 us, 270 with four pieces and 352 threads, 300 with eight and 192.
static int norm8_bwd_pieces(int n) { return n <= 2048 ? 1 : n <= 8192 ? 2 : 8; }
static int norm8_bwd_threads(int n) {
  const int per_warp = 32 * norm8_bwd_pieces(n);
  if (n > 8192) return 256;
  return (n / 8 + per_warp - 1) / per_warp * 32;
}
extern "C" int ody_rmsnorm8_bwd_blocks(int64_t rows, int n) {
  const int per_sm = (n > 8192 ? 256 : 600) / norm8_bwd_threads(n);
  const int64_t b = 148 * (per_sm < 16 ? per_sm : 16);
  return (int)(rows < b ? (rows > 0 ? rows : 1) : b);
}

template <int FMT, int NP, int STAGES, int THREADS, int BLOCKS>
static int launch_norm8_bwd(const void* dy, const void* codes, const float* scales, const void* w, const float* rstd, const void* ds,
                            void* dx, float* dw_partial, int64_t rows, int n, int nb, cudaStream_t st) {
  static std::atomic<uint64_t> done{0};
  const int e = allow_smem(rmsnorm8_bwd_k<FMT, NP, STAGES, THREADS, BLOCKS>, STAGES * NP * THREADS * Stage<NP>::BYTES, done);
  if (e) return e;
  const int threads = norm8_bwd_threads(n);
  return launch_kernel(rmsnorm8_bwd_k<FMT, NP, STAGES, THREADS, BLOCKS>, nb, threads, STAGES * NP * threads * Stage<NP>::BYTES, st, 1, (const bf16*)dy,
                       (const uint8_t*)codes, scales, (const bf16*)w, rstd, (const bf16*)ds, (bf16*)dx, dw_partial, rows, n);
}

extern "C" int ody_rmsnorm8_bwd(const void* dy, const void* codes, const float* scales, const void* w, const float* rstd, const void* ds,
                                void* dx, void* dw, int dw_bf16, float* dw_partial, int64_t rows, int n, int fmt, cudaStream_t st) {
  if (bad_rows(rows, n, fmt) || n > ODY_RMSNORM8_MAX || !aligned(dy, 16) || !aligned(ds, 16) || !aligned(w, 16) || !aligned(dx, 16) ||
      !aligned(codes, 8) || !aligned(dw_partial, 16))
    return (int)cudaErrorInvalidValue;
  const int nb = ody_rmsnorm8_bwd_blocks(rows, n);
  int e;
#define R(...)                                                                                                             \
  e = fmt == E4M3 ? launch_norm8_bwd<E4M3, __VA_ARGS__>(dy, codes, scales, w, rstd, ds, dx, dw_partial, rows, n, nb, st)     \
                  : launch_norm8_bwd<INT8, __VA_ARGS__>(dy, codes, scales, w, rstd, ds, dx, dw_partial, rows, n, nb, st)
  if (n <= 2048) R(1, 4, 256, 2); else if (n <= 4096) R(2, 4, 256, 2); else if (n <= 8192) R(2, 4, 512, 1); else R(8, 2, 256, 1);
#undef R
  if (e) return e;
  return ody_colsum(dw_partial, dw, dw_bf16, nb, n, st);
}
