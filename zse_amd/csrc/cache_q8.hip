// A key-value cache in 8 bits: written as keys are rotated, read back into pages of the compute type, and attended to by
// single tokens.
//
// A head's channels of one token are 8-bit codes and one float scale, keys and values apart:
//   a = max |x_c|,  scale = a / top,  code_c = round(x_c * (top / a)),  value = code_c * scale
// with top = 127 and whole numbers (format 0, int8), or top = 448 and the 8-bit floats of four exponent and three
// mantissa bits without infinities (format 1, e4m3), ties to even.  a < 2^-100 counts as zero (scale 0, codes 0).  A head
// with a value that is not finite has scale NaN and codes 0: whoever sees the key gets NaN.
//
// Layout: [page][key head][page size / 16][blocks of 64 channels] of 1,024 bytes, the last block filled up with zeros.
// Keys: [16 tokens][64 channels].  Values: [4][16][4][4], token 4 a + d and channel 16 c + b of the block at [a][b][c][d],
// so that the 16 bytes that one lane loads are four output channels' operands for four neighbouring keys, and a wave's load
// is a whole block of either.  Scales: [page][key head][keys, values][page size].
#include "common.h"
#include "packed_call.h"

#include <algorithm>
#include <cfloat>
#include <type_traits>

extern "C" int zk_steplist_register(const char* name, int nargs, void* fn);
#define ZK_ENTER(fn) \
  static const int fn##_entered = zk_steplist_register(#fn, zk_packed::Call<fn>::nargs, (void*)zk_packed::Call<fn>::call);

#define Q8_PIECE 16           // tokens of a piece
#define Q8_BLOCK 64           // channels of a block
#define Q8_BYTES 1024         // of a block of a piece

__host__ __device__ __forceinline__ int q8_blocks(int hd) { return (hd + Q8_BLOCK - 1) / Q8_BLOCK; }
__device__ __forceinline__ int q8_key_at(int t, int c) { return t * 64 + c; }
__device__ __forceinline__ int q8_value_at(int t, int c) { return (t / 4) * 256 + (c % 16) * 16 + (c / 16) * 4 + t % 4; }

// The first byte of a head's piece of 16 tokens.
__device__ __forceinline__ size_t q8_piece(int page, int piece, int head, int nkv, int pieces, int blocks) {
  return (((size_t)page * nkv + head) * pieces + piece) * (size_t)(blocks * Q8_BYTES);
}
__device__ __forceinline__ size_t q8_scale(int page, int head, int nkv, int bs, int values) {
  return (((size_t)page * nkv + head) * 2 + values) * (size_t)bs;
}

// x / n; ``shift``: where n is a power of two its exponent, else -1 (a division is some thirty instructions, and a kernel of few
// blocks is as long as one wave's chain of them).
__device__ __forceinline__ int q8_div(int x, int n, int shift) { return shift >= 0 ? x >> shift : x / n; }
static int q8_shift(int n) { return (n & (n - 1)) == 0 ? __builtin_ctz(n) : -1; }

template <int FMT>
__device__ __forceinline__ float q8_top() { return FMT == 0 ? 127.f : 448.f; }

// Four values times ``factor`` as four codes.  |x| factor is at most top and a rounding, which the nearest code of either kind is top
// for: nothing has to be cut off.
template <int FMT>
__device__ __forceinline__ unsigned q8_codes(const float (&x)[4], float factor) {
#ifdef __HIP_DEVICE_COMPILE__
  if constexpr (FMT == 0) {
    unsigned w[4];                    // 1.5 * 2^23 + a whole number: its two's complement in the lowest byte
#pragma unroll
    for (int e = 0; e < 4; e++) w[e] = __float_as_uint(__fmaf_rn(x[e], factor, 12582912.f));
    const unsigned lo = __builtin_amdgcn_perm(w[1], w[0], 0x0c0c0400), hi = __builtin_amdgcn_perm(w[3], w[2], 0x04000c0c);
    return lo | hi;
  } else {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0] * factor, x[1] * factor, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x[2] * factor, x[3] * factor, lo, true);
  }
#else
  return 0;
#endif
}

// Scale and factor of a head whose largest magnitude is ``a`` (NaN or infinity where a value is not finite).
template <int FMT>
__device__ __forceinline__ void q8_scales(float a, float& scale, float& factor) {
  const float top = q8_top<FMT>();
  if (!(a <= FLT_MAX)) {
    scale = __int_as_float(0x7fc00000);
    factor = 0.f;
  } else if (a < 0x1p-100f) {
    scale = factor = 0.f;
  } else {
    scale = __fmul_rn(a, 1.f / top);
    factor = __fdiv_rn(top, a);
  }
}

// Sine and cosine of pos * freq, positions below 2^24.  The product is held in two floats (rounded to one it is off by up to half
// a step of the angle, 2^-12 at position 4,096 and 2^-7 at 131,072), less whole quarters of a turn (pi / 2 in two floats; n times the
// first takes nothing from a multiple of its last place), then one float r and what that leaves, which turns the result to first
// order.  |r| is at most pi / 4 (and a rounding): the Taylor sums up to r^9 and r^10 are off by less than 2e-9.
__device__ __forceinline__ void q8_sincos(float pos, float freq, float& sn, float& cs) {
  const float angle = __fmul_rn(pos, freq), low = __fmaf_rn(pos, freq, -angle);
  float n = rintf(angle * 0.63661977f);
  float a = __fmaf_rn(n, -1.57079637f, angle), b = __fmaf_rn(n, 4.37113883e-8f, low);
  n += rintf((a + b) * 0.63661977f);                 // (of large angles the first count is a quarter or two off)
  a = __fmaf_rn(n, -1.57079637f, angle);
  b = __fmaf_rn(n, 4.37113883e-8f, low);
  const float r = a + b, part = r - a, rest = (a - (r - part)) + (b - part);
  const float r2 = r * r, half = 0.5f * r2, one = 1.f - half;
  const float s0 = __fmaf_rn(r * r2, __fmaf_rn(r2, __fmaf_rn(r2, __fmaf_rn(r2, 1.f / 362880.f, -1.f / 5040.f), 1.f / 120.f), -1.f / 6.f), r);
  const float c4 = __fmaf_rn(r2, __fmaf_rn(r2, __fmaf_rn(r2, -1.f / 3628800.f, 1.f / 40320.f), -1.f / 720.f), 1.f / 24.f);
  const float c0 = one + __fmaf_rn(r2 * r2, c4, (1.f - one) - half);
  const float s = __fmaf_rn(c0, rest, s0), c = __fmaf_rn(s0, -rest, c0);
  const int quarter = (int)n;
  sn = quarter & 1 ? c : s;
  cs = quarter & 1 ? s : c;
  if (quarter & 2) sn = -sn;
  if ((quarter + 1) & 2) cs = -cs;
}

typedef float q8_f4 __attribute__((ext_vector_type(4)));
typedef unsigned q8_u4 __attribute__((ext_vector_type(4)));
typedef act_t q8_a4 __attribute__((ext_vector_type(4)));
typedef act_t q8_a8 __attribute__((ext_vector_type(8)));
#if ZSE_ACT_BF16
typedef __bf16 q8_b8 __attribute__((ext_vector_type(8)));
#endif

// Four codes as four numbers of the type that the products take.
template <int FMT>
__device__ __forceinline__ void q8_floats(unsigned codes, float (&x)[4]) {
#ifdef __HIP_DEVICE_COMPILE__
  if constexpr (FMT == 0) {
    x[0] = (float)(int)(int8_t)codes;
    x[1] = (float)(int)(int8_t)(codes >> 8);
    x[2] = (float)(int)(int8_t)(codes >> 16);
    x[3] = (float)((int)codes >> 24);
  } else {
    x[0] = __builtin_amdgcn_cvt_f32_fp8((int)codes, 0);
    x[1] = __builtin_amdgcn_cvt_f32_fp8((int)codes, 1);
    x[2] = __builtin_amdgcn_cvt_f32_fp8((int)codes, 2);
    x[3] = __builtin_amdgcn_cvt_f32_fp8((int)codes, 3);
  }
#endif
}

// ---------------------------------------------------------------- written
// A block takes four rows of the step, a group of LANES lanes a head of them at a time, four neighbouring channels a lane: the
// head's largest magnitude is a maximum over the group's lanes, and four rows whose slots are four in a row from a multiple of four on
// (a portion's) leave their values as whole words of the layout.  Such fours are taken together wherever they begin; the rows that
// are in none (single tokens, a portion's ends) are taken as they come.  Sines and cosines of the four rows are worked out once, in LDS.
// The channels that a lane's turn with come from the lane that has them, not from memory (4,092 rows as below 36.3 -> 33.0 us; 64 rows of
// 16 heads of 256 out of three planes 7.2 -> 5.8, with the planes asked for together, out of six 8.7 -> 6.3).  The first moves
// 3.6 TB/s, with 1.22 M write requests for 0.79 M lines of 64 bytes (values': four bytes a store at a stride of 16); one wave's chain of waits
// bounds the others; 72 registers instead of 80, for a seventh wave a SIMD, spill (36.6).
template <bool SUMS>
struct Q8Rows {
  const act_t* rows;
  const float* planes;        // partial sums of a split product
  int ld, sums;
  size_t plane;
  __device__ __forceinline__ act_t at(int row, unsigned i) const {
    if constexpr (!SUMS) return (rows + (size_t)row * ld)[i];
    const float* r = planes + (size_t)row * ld;
    float x = r[i];
    for (int p = 1; p < sums; p++) x += (r + p * plane)[i];
    return from_f32<act_t>(x);
  }
  // four values of four rows; of planes three at a time, so that a turn is one wait for twelve loads (the last again where fewer are left)
  __device__ __forceinline__ void at4(const int (&row)[4], unsigned i, q8_a4 (&to)[4]) const {
    if constexpr (!SUMS) {
#pragma unroll
      for (int t = 0; t < 4; t++) to[t] = *(const q8_a4*)(rows + (size_t)row[t] * ld + i);
    } else {
      q8_f4 x[4];
      for (int p = 0; p < sums; p += 3) {
        q8_f4 y[3][4];
#pragma unroll
        for (int u = 0; u < 3; u++)
#pragma unroll
          for (int t = 0; t < 4; t++) y[u][t] = *(const q8_f4*)(planes + min(p + u, sums - 1) * plane + (size_t)row[t] * ld + i);
#pragma unroll
        for (int t = 0; t < 4; t++) {
          x[t] = p == 0 ? y[0][t] : x[t] + y[0][t];
          if (p + 1 < sums) x[t] += y[1][t];
          if (p + 2 < sums) x[t] += y[2][t];
        }
      }
#pragma unroll
      for (int t = 0; t < 4; t++) to[t] = q8_a4{from_f32<act_t>(x[t][0]), from_f32<act_t>(x[t][1]), from_f32<act_t>(x[t][2]), from_f32<act_t>(x[t][3])};
    }
  }
};

template <bool SUMS>
struct Q8Write {
  Q8Rows<SUMS> from;
  act_t* q_out;
  const int *positions, *slot_map;
  const float* inv_freq;
  uint8_t *kcodes, *vcodes;
  float* scales;
  int ldq, rotary_dim, T, nh, nkv, hd, bs, bs_shift, num_pages, heads;
};

// The largest of a group of 16, 32 or 64 lanes' magnitudes as bits (a NaN is larger than infinity, and that than any number).
template <int LANES>
__device__ __forceinline__ float q8_largest(float v) {
  auto larger = [](float a, float b) { return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b))); };
  float a = v, b = v;
  if constexpr (LANES > 32) {
    wave_pair32(v, a, b);
    v = larger(a, b);
  }
  if constexpr (LANES > 16) {
    wave_pair16(v, a, b);
    v = larger(a, b);
  }
  v = larger(v, wave_dpp<ZSE_DPP_ROR8>(v));
  v = larger(v, wave_dpp<ZSE_DPP_ROR4>(v));
  v = larger(v, wave_dpp<ZSE_DPP_XOR2>(v));
  return larger(v, wave_dpp<ZSE_DPP_XOR1>(v));
}

// Another lane's four values.
__device__ __forceinline__ q8_a4 q8_of_lane(q8_a4 x, int lane) {
#ifdef __HIP_DEVICE_COMPILE__
  typedef int words __attribute__((ext_vector_type(sizeof(q8_a4) / 4)));
  words w = __builtin_bit_cast(words, x);
#pragma unroll
  for (int i = 0; i < (int)(sizeof(q8_a4) / 4); i++) w[i] = __builtin_amdgcn_ds_bpermute(lane * 4, w[i]);
  return __builtin_bit_cast(q8_a4, w);
#else
  return x;
#endif
}

// WHOLE: rows, heads and half the rotation are whole fours at addresses of whole fours.
template <int FMT, int LANES, bool WHOLE, bool SUMS>
__global__ __launch_bounds__(256, WHOLE ? (SUMS ? 3 : 4) : 2) void write_q8_kernel(Q8Write<SUMS> p) {
#ifdef __HIP_DEVICE_COMPILE__
  constexpr int HEADS = 256 / LANES;                // of a pass
  __shared__ q8_f4 s_sin[4][32], s_cos[4][32];
  const int lane = threadIdx.x & 63, sub = threadIdx.x / LANES, c0 = threadIdx.x % LANES * 4, half = p.rotary_dim / 2;
  const int blocks = q8_blocks(p.hd), pieces = p.bs / Q8_PIECE, t0 = blockIdx.x * 4;
  const bool rotated = c0 < p.rotary_dim, low = c0 < half, padded = c0 >= blocks * Q8_BLOCK;
  // where a lane's channels lie in a head (lanes without any read the head's first), and the lane that has those that they turn with
  const int own = c0 < p.hd ? c0 : 0, mate_lane = !rotated ? lane : low ? lane + half / 4 : lane - half / 4;
  const int turn_at = rotated ? (low ? c0 : c0 - half) / 4 : 0;
  const int key_at = c0 / Q8_BLOCK * Q8_BYTES + c0 % Q8_BLOCK, value_at = c0 / Q8_BLOCK * Q8_BYTES + q8_value_at(0, c0 % Q8_BLOCK);
  const unsigned sign = low ? 0x80000000u : 0u;             // a - b turns where the lane holds the pair's first
  const unsigned head_bytes = pieces * blocks * Q8_BYTES;
  // lane i: the slot of row t0 - 3 + i, for ten rows; bit i of ``fours``: rows i to i + 3 are such a four
  const int near = t0 - 3 + lane;
  int slots = p.slot_map && lane < 10 && near >= 0 && near < p.T ? p.slot_map[near] : -1;
  const float position = lane < 10 && near >= 0 && near < p.T ? (float)p.positions[near] : 0.f;
  const int page = q8_div(slots, p.bs, p.bs_shift);
  if (page >= p.num_pages) slots = -1;
  const int off = slots - page * p.bs;
  // (what follows is of a slot that is there; of others it is not used)
  const int piece_of = slots < 0 ? 0 : page * p.nkv * pieces + off / Q8_PIECE, scale_of = slots < 0 ? 0 : page * p.nkv * 2 * p.bs + off;
  const int s1 = __shfl(slots, lane + 1), s2 = __shfl(slots, lane + 2), s3 = __shfl(slots, lane + 3);
  const unsigned fours = (unsigned)__ballot(lane < 7 && slots >= 0 && slots % 4 == 0 && s1 == slots + 1 && s2 == slots + 2 && s3 == slots + 3);
  for (int taken = 0; taken < 2; taken++) {
    // the four that begins among the block's rows, then the block's rows that are in none
    const bool four = taken == 0;
    const unsigned held = (1u << min(4, p.T - t0)) - 1;       // the block's rows that there are
    const unsigned mine = four ? (fours & 0x78 ? 15 : 0)
                               : held & ~(fours | fours >> 1 | fours >> 2 | fours >> 3);      // bit t: there is a row t
    if (!mine) continue;
    const int start = four ? __builtin_ctz(fours & 0x78) : 3;
    int row[4], slot[4], at[4];
    size_t piece[4];
#pragma unroll
    for (int t = 0; t < 4; t++) {
      row[t] = min(t0 - 3 + start + t, p.T - 1);              // (one that is not there is not stored)
      slot[t] = mine >> t & 1 ? __builtin_amdgcn_readlane(slots, start + t) : -1;
      at[t] = __builtin_amdgcn_readlane(off, start + t) % Q8_PIECE;
      piece[t] = (size_t)__builtin_amdgcn_readlane(piece_of, start + t) * (unsigned)(blocks * Q8_BYTES);
    }
    // lane t of every quad: row t's, for its scales
    const int quad_of = __shfl(slots, start + (lane & 3)), quad_scale = __shfl(scale_of, start + (lane & 3));
    const int quad_slot = mine >> (lane & 3) & 1 ? quad_of : -1;
    const bool stores = slot[0] >= 0 || slot[1] >= 0 || slot[2] >= 0 || slot[3] >= 0;
    bool turned = false;
    const int pass = gridDim.y * HEADS;
    q8_a4 xr[4], yr[4];                              // a row's four channels, and those that they turn with: a pass ahead
    auto ask = [&](int base) {
      const unsigned head_at = min(base + sub, p.heads - 1) * p.hd;
      if constexpr (WHOLE) {
        p.from.at4(row, head_at + own, xr);
      } else {
#pragma unroll
        for (int t = 0; t < 4; t++) {
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int c = c0 + e, mate = c >= p.rotary_dim ? c : c < half ? c + half : c - half;
            xr[t][e] = p.from.at(row[t], head_at + (c < p.hd ? c : 0));
            yr[t][e] = p.from.at(row[t], head_at + (c < p.hd ? mate : 0));
          }
        }
      }
    };
    ask(blockIdx.y * HEADS);
    for (int base = blockIdx.y * HEADS; base < p.heads; base += pass) {
      const int head = min(base + sub, p.heads - 1);
      const bool live = base + sub < p.heads, is_q = head < p.nh, is_v = head >= p.nh + p.nkv;
      if (!turned && half > 0 && base < p.nh + p.nkv) {        // the first pass with queries or keys
        if (taken) __syncthreads();                            // (the other rows' angles have been read)
        // a row a wave, so that all four are worked out side by side
        const int t = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        if (mine >> t & 1) {
          const float pos = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(position), start + t));
          for (int i = lane; i < half; i += 64) q8_sincos(pos, p.inv_freq[i], ((float*)s_sin[t])[i], ((float*)s_cos[t])[i]);
        }
        __syncthreads();
        turned = true;
      }
      float x[4][4], y[4][4];
      if constexpr (WHOLE) {
        if (half > 0 && base < p.nh + p.nkv) {
#pragma unroll
          for (int t = 0; t < 4; t++) yr[t] = q8_of_lane(xr[t], mate_lane);
        }
      }
#pragma unroll
      for (int t = 0; t < 4; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          x[t][e] = to_f32(xr[t][e]);
          y[t][e] = to_f32(yr[t][e]);
          if (WHOLE) y[t][e] = __uint_as_float(__float_as_uint(y[t][e]) ^ sign);
        }
      if (base + pass < p.heads) ask(base + pass);
      if (!is_v) {
#pragma unroll
        for (int t = 0; t < 4; t++) {
          if constexpr (WHOLE) {
            if (rotated) {
              const q8_f4 sn = s_sin[t][turn_at], cs = s_cos[t][turn_at];
#pragma unroll
              for (int e = 0; e < 4; e++) x[t][e] = __fmaf_rn(x[t][e], cs[e], __fmul_rn(y[t][e], sn[e]));        // as rotate_pair
            }
          } else {
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const int c = c0 + e;
              if (c >= p.rotary_dim) continue;
              const bool first = c < half;
              const int i = first ? c : c - half;
              const float sn = ((const float*)s_sin[t])[i], cs = ((const float*)s_cos[t])[i];
              x[t][e] = __fmaf_rn(x[t][e], cs, __fmul_rn(y[t][e], first ? -sn : sn));
            }
          }
        }
      }
      if (is_q && live) {
#pragma unroll
        for (int t = 0; t < 4; t++) {
          if (!(mine >> t & 1)) continue;
          act_t* to = p.q_out + (size_t)row[t] * p.ldq + (unsigned)(head * p.hd + c0);
          if constexpr (WHOLE) {
            if (c0 < p.hd) *(q8_a4*)to = q8_a4{from_f32<act_t>(x[t][0]), from_f32<act_t>(x[t][1]), from_f32<act_t>(x[t][2]), from_f32<act_t>(x[t][3])};
          } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
              if (c0 + e < p.hd) to[e] = from_f32<act_t>(x[t][e]);
          }
        }
      }
      if (!stores || base + HEADS <= p.nh) continue;           // (all lanes of the block alike)
      float most[4];
#pragma unroll
      for (int t = 0; t < 4; t++) {
        if constexpr (WHOLE) {
          if (c0 >= p.hd) x[t][0] = x[t][1] = x[t][2] = x[t][3] = 0.f;          // the last block is filled up with zeros
        } else {
#pragma unroll
          for (int e = 0; e < 4; e++)
            if (c0 + e >= p.hd) x[t][e] = 0.f;
        }
        const float a = __builtin_elementwise_maximum(__builtin_elementwise_maximum(fabsf(x[t][0]), fabsf(x[t][1])), fabsf(x[t][2]));
        most[t] = q8_largest<LANES>(__builtin_elementwise_maximum(a, fabsf(x[t][3])));
      }
      // a lane works out one row's factor for the four lanes of its quad
      float scale, factor;
      q8_scales<FMT>(lane & 2 ? (lane & 1 ? most[3] : most[2]) : (lane & 1 ? most[1] : most[0]), scale, factor);
      const float factors[4] = {wave_dpp<0x00>(factor), wave_dpp<0x55>(factor), wave_dpp<0xAA>(factor), wave_dpp<0xFF>(factor)};
      unsigned word[4];                                // a row's four codes
#pragma unroll
      for (int t = 0; t < 4; t++) {
        if (factors[t] == 0.f) {                       // nothing that a code could hold, or a value that is not finite
#pragma unroll
          for (int e = 0; e < 4; e++) x[t][e] = 0.f;
        }
        word[t] = q8_codes<FMT>(x[t], factors[t]);
      }
      if (is_q || !live) continue;
      const int kvh = (head - p.nh) - (is_v ? p.nkv : 0);
      const unsigned head_at = kvh * head_bytes;
      if (padded) {
      } else if (!is_v) {
#pragma unroll
        for (int t = 0; t < 4; t++)
          if (slot[t] >= 0) *(unsigned*)(p.kcodes + piece[t] + at[t] * 64 + (head_at + key_at)) = word[t];
      } else if (four) {
        // the four rows' bytes of a channel side by side
        const unsigned a = __builtin_amdgcn_perm(word[1], word[0], 0x05010400), b = __builtin_amdgcn_perm(word[1], word[0], 0x07030602);
        const unsigned d = __builtin_amdgcn_perm(word[3], word[2], 0x05010400), f = __builtin_amdgcn_perm(word[3], word[2], 0x07030602);
        uint8_t* to = p.vcodes + piece[0] + at[0] * 64 + (head_at + value_at);          // (the next channel: 16 bytes on)
        *(unsigned*)to = __builtin_amdgcn_perm(d, a, 0x05040100);
        *(unsigned*)(to + 16) = __builtin_amdgcn_perm(d, a, 0x07060302);
        *(unsigned*)(to + 32) = __builtin_amdgcn_perm(f, b, 0x05040100);
        *(unsigned*)(to + 48) = __builtin_amdgcn_perm(f, b, 0x07060302);
      } else {
#pragma unroll
        for (int t = 0; t < 4; t++) {
          if (slot[t] < 0) continue;
          uint8_t* to = p.vcodes + piece[t] + (at[t] / 4 * 256 + at[t] % 4) + (head_at + value_at);
#pragma unroll
          for (int e = 0; e < 4; e++) to[16 * e] = (uint8_t)(word[t] >> (8 * e));
        }
      }
      // the head's first four lanes: a row's scale each
      if (c0 < 16 && quad_slot >= 0) p.scales[(unsigned)quad_scale + (size_t)(2 * kvh + is_v) * p.bs] = scale;
    }
  }
#endif
}

// ---------------------------------------------------------------- read back
// A wave reads a piece of one head, or two neighbouring ones (PAIRS: pages of an even number of pieces): keys eight channels a lane, so
// that a load is 512 bytes in a row and a store whole rows of 64 channels; values as the layout has them, four neighbouring tokens of
// four channels a lane.  Where they go out transposed in 16 bits, rows of 16 lanes exchange words, and a lane stores eight neighbouring
// tokens of a channel: with pairs a store is 16 channels' runs of 64 bytes.
struct Q8Read {
  const uint8_t *kcodes, *vcodes;
  const float* scales;
  const int *block_table, *q_start, *ctx_len;
  act_t *k, *v;
  int R, max_blocks, max_ctx, window, nkv, hd, bs, bs_shift, num_pages;
};

template <int FMT, bool TRANSPOSED, bool WHOLE, bool PAIRS>
__global__ __launch_bounds__(256) void read_q8_kernel(Q8Read p) {
#ifdef __HIP_DEVICE_COMPILE__
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  constexpr int U = PAIRS ? 2 : 1;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), pieces = p.bs / Q8_PIECE;
  const int turns = pieces / U, turns_shift = p.bs_shift >= 0 ? p.bs_shift - 4 - (U - 1) : -1, per_page = turns * p.nkv;
  // the requests' pages are numbered through, 64 requests at a time: lane i knows where those of request r0 + i end
  int r0 = -64, before = 0, upto = 0, ends = 0, ctx_of = 0, first_of = 0;      // before, upto: of the 64 requests' pages
  for (int item = blockIdx.x * 4 + wave;; item += gridDim.x * 4) {
    const int x = item / per_page, rest = item - x * per_page;
    const int head = q8_div(rest, turns, turns_shift), sub = (rest - head * turns) * U;
    while (x >= upto) {
      r0 += 64;
      if (r0 >= p.R) return;
      const int r = min(r0 + lane, p.R - 1), ctx = min(p.ctx_len[r], p.max_ctx), rows = p.q_start ? p.q_start[r + 1] - p.q_start[r] : 1;
      ctx_of = ctx;
      first_of = q8_div(p.window > 0 ? max(0, ctx - rows + 1 - p.window) : 0, p.bs, p.bs_shift);
      ends = upto + wave_running_sum(r0 + lane < p.R ? max(0, q8_div(max(ctx, 0) + p.bs - 1, p.bs, p.bs_shift) - first_of) : 0);
      before = upto;
      upto = __builtin_amdgcn_readlane(ends, 63);
    }
    const int of = __ffsll(__ballot(ends > x)) - 1, r = r0 + of;
    const int ctx = __builtin_amdgcn_readlane(ctx_of, of);
    const int j = __builtin_amdgcn_readlane(first_of, of) + x - (of ? __builtin_amdgcn_readlane(ends, of - 1) : before);
    const int page = p.block_table[(size_t)r * p.max_blocks + j], i = j * pieces + sub;
    if (page < 0 || page >= p.num_pages) continue;
    const int there = ctx - i * Q8_PIECE, blocks = q8_blocks(p.hd);      // tokens that are there: below 1, none
    const size_t at = q8_piece(page, sub, head, p.nkv, pieces, blocks);
    const float* scales = p.scales + q8_scale(page, head, p.nkv, p.bs, 0) + sub * Q8_PIECE;
    const size_t out = ((size_t)page * p.nkv + head) * (size_t)(p.bs * p.hd);
    const int t0 = lane / 8, c8 = lane % 8 * 8, row = lane / 16, col = lane % 16;
    float ks[2 * U];
#pragma unroll
    for (int u = 0; u < 2 * U; u++) ks[u] = scales[t0 + 8 * u];
    constexpr bool EIGHTS = TRANSPOSED && sizeof(act_t) == 2;
    static_assert(EIGHTS || !PAIRS, "pairs of pieces go out by eights");
    // the tokens that a lane stores of a channel: eight from ``first``, or four
    const int first = PAIRS ? (row & 1) * 16 + row / 2 * 8 : row / 2 * 8;
    q8_f4 vs[2];
    vs[0] = *(const q8_f4*)(scales + p.bs + (EIGHTS ? first : row * 4));
    vs[1] = *(const q8_f4*)(scales + p.bs + (EIGHTS ? first + 4 : row * 4));
    for (int n = 0; n < blocks; n++) {
      u2 kw[2 * U];
      q8_u4 vw[U];
#pragma unroll
      for (int u = 0; u < 2 * U; u++)
        kw[u] = *(const u2*)(p.kcodes + at + (size_t)(u / 2) * blocks * Q8_BYTES + n * Q8_BYTES + u % 2 * 512 + lane * 8);
#pragma unroll
      for (int u = 0; u < U; u++) vw[u] = *(const q8_u4*)(p.vcodes + at + (size_t)u * blocks * Q8_BYTES + n * Q8_BYTES + lane * 16);
#pragma unroll
      for (int u = 0; u < 2 * U; u++) {
        const int t = t0 + 8 * u, c = n * Q8_BLOCK + c8;
        float lo[4], hi[4];
        q8_floats<FMT>(kw[u][0], lo);
        q8_floats<FMT>(kw[u][1], hi);
        q8_a8 x;
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = from_f32<act_t>(t < there ? (e < 4 ? lo[e] : hi[e - 4]) * ks[u] : 0.f);
        act_t* to = p.k + out + (size_t)(sub * Q8_PIECE + t) * p.hd + c;
        if constexpr (WHOLE) {
          if (c < p.hd) *(q8_a8*)to = x;
        } else {
#pragma unroll
          for (int e = 0; e < 8; e++)
            if (c + e < p.hd) to[e] = x[e];
        }
      }
      if constexpr (EIGHTS) {
        // Odd rows of the first word change places with even rows of the second: row 0 has the first word's tokens 0 to 7, row 2 its
        // tokens 8 to 15, rows 1 and 3 the second's.  The second word: the same channels' of the other piece, or the next 16 channels'.
#pragma unroll
        for (int b = 0; b < 4; b += PAIRS ? 1 : 2) {
          const auto w = __builtin_amdgcn_permlane16_swap(vw[0][b], PAIRS ? vw[U - 1][b] : vw[0][(b + 1) % 4], false, false);
          const int c = n * Q8_BLOCK + 16 * (PAIRS ? b : b + (row & 1)) + col;
          float lo[4], hi[4];
          q8_floats<FMT>(w[0], lo);
          q8_floats<FMT>(w[1], hi);
          q8_a8 y;
#pragma unroll
          for (int e = 0; e < 8; e++) y[e] = from_f32<act_t>(first + e < there ? (e < 4 ? lo[e] : hi[e - 4]) * vs[e / 4][e % 4] : 0.f);
          if (c < p.hd) *(q8_a8*)(p.v + out + (size_t)c * p.bs + sub * Q8_PIECE + first) = y;
        }
      } else {
#pragma unroll
        for (int b = 0; b < 4; b++) {
          const int c = n * Q8_BLOCK + 16 * b + col, t = row * 4;
          float x[4];
          q8_floats<FMT>(vw[0][b], x);
          q8_a4 y;
#pragma unroll
          for (int e = 0; e < 4; e++) y[e] = from_f32<act_t>(t + e < there ? x[e] * vs[0][e] : 0.f);
          if (c < p.hd) {
            if constexpr (TRANSPOSED) *(q8_a4*)(p.v + out + (size_t)c * p.bs + sub * Q8_PIECE + t) = y;
            else {
#pragma unroll
              for (int e = 0; e < 4; e++) p.v[out + (size_t)(sub * Q8_PIECE + t + e) * p.hd + c] = y[e];
            }
          }
        }
      }
    }
  }
#endif
}

// ---------------------------------------------------------------- attended to
// Scores and outputs by 16 x 16 matrix products whose columns are the query heads of one key head (16 at a time) and whose rows
// are keys, then channels: S = K Q' over channels, O' = V' P over keys.  A lane of S holds four neighbouring keys of one head,
// and that is the operand that O' takes: weights stay in registers.  Codes are whole in bfloat16 (8 bits of mantissa), so a
// key's scale multiplies its score, a value's scale its weight.
//
// A block (four waves) takes a chunk of keys at absolute positions, a wave pairs of pieces of 16 in turn; the running maximum, the
// sum and O' of the four waves are joined in LDS, the chunks' results by a second kernel.  The chunk follows from the width
// of the table alone, so that a request's sums are cut alike whoever shares its step.
struct Q8Attention {
  const act_t* q;
  const uint8_t *kcodes, *vcodes;
  const float* scales;
  const int *block_table, *ctx_len;
  act_t* out;
  float *part_o, *part_ml;          // [R][nh][splits][channels, filled up] and [..][2]
  int q_stride, max_blocks, max_ctx, nh, nkv, hd, pieces, pieces_shift, num_pages, window, chunk, chunk_shift, q_whole;
  float k1, k2, c2;                 // z log2(e) = k1 dot, or c2 tanh(k2 dot)
  float rest;                       // what k1, or c2, is short of its value
};

#if ZSE_ACT_BF16
template <int FMT>
__device__ __forceinline__ void q8_halves(unsigned codes, unsigned& lo, unsigned& hi) {
#ifdef __HIP_DEVICE_COMPILE__
  if constexpr (FMT == 0) {
    float x[4];                       // whole numbers up to 127: the upper halves hold them
    q8_floats<FMT>(codes, x);
    lo = __builtin_amdgcn_perm(__float_as_uint(x[1]), __float_as_uint(x[0]), 0x07060302);
    hi = __builtin_amdgcn_perm(__float_as_uint(x[3]), __float_as_uint(x[2]), 0x07060302);
  } else {
    lo = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.f, false));
    hi = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, 1.f, true));
  }
#endif
}
template <int FMT>
__device__ __forceinline__ q8_b8 q8_operand(unsigned a, unsigned b) {
  q8_u4 w;
  unsigned lo = 0, hi = 0;
  q8_halves<FMT>(a, lo, hi);
  w[0] = lo;
  w[1] = hi;
  q8_halves<FMT>(b, lo, hi);
  w[2] = lo;
  w[3] = hi;
  return __builtin_bit_cast(q8_b8, w);
}
#endif

template <int FMT, int NB, bool CAP, bool DIRECT, bool ONCE>
__global__ __launch_bounds__(256, 2) void attention_q8_kernel(Q8Attention p) {
#ifdef __HIP_DEVICE_COMPILE__
  extern __shared__ float s_join[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), col = lane & 15, g = lane >> 4;
  // Chunks are the slowest index, the one that the window cuts the last: what is left for a last round of blocks is chunks that
  // requests have little of (64 requests of 200 to 3,840 keys 56.2 -> 55.1 us, eight of 8,192 48.6 -> 47.3; with chunks as the fastest
  // index and eight of them a request, an XCD had the same chunk of all requests: 74 us).  Neighbouring blocks go to different
  // XCDs: requests are turned by the chunk, so that none has one request alone.
  const int splits = gridDim.z, split = p.window > 0 ? (blockIdx.z + 1) % splits : blockIdx.z, r = (blockIdx.y + blockIdx.z) % gridDim.y;
  const int group = p.nh / p.nkv, kvh = blockIdx.x % p.nkv, head0 = blockIdx.x / p.nkv * 16, heads = min(16, group - head0);
  // without a window the chunk's place in the table does not wait for the request's length
  int early = -1;
  if (p.window == 0 && p.max_ctx > 0) early = p.block_table[(size_t)r * p.max_blocks + min(q8_div(split * (p.chunk / Q8_PIECE) + lane, p.pieces, p.pieces_shift), p.max_blocks - 1)];
  const int ctx = min(p.ctx_len[r], p.max_ctx), first = p.window > 0 ? max(0, ctx - p.window) : 0;
  const int from = ((first >> p.chunk_shift) + split) << p.chunk_shift;
  const int begin = max(first, from), end = min(ctx, from + p.chunk);
  const int head = kvh * group + head0 + col;             // this lane's column, if col < heads
  if (begin >= end) {
    if (DIRECT)
      for (int i = threadIdx.x; i < heads * p.hd; i += 256)
        p.out[((size_t)r * p.nh + kvh * group + head0) * p.hd + i] = from_f32<act_t>(0.f);
    return;
  }
  // lane i: where the chunk's piece i lies; -1 where the table names no page
  const int p0 = begin / Q8_PIECE, n_pieces = (end + Q8_PIECE - 1) / Q8_PIECE - p0;
  int piece_at = -1, scale_at = 0;
  if (lane < n_pieces) {
    const int i = p0 + lane, of = q8_div(i, p.pieces, p.pieces_shift), sub = i - of * p.pieces;
    const int page = p.window == 0 ? early : p.block_table[(size_t)r * p.max_blocks + of];
    if (page >= 0 && page < p.num_pages) {
      const int at = page * p.nkv + kvh;
      piece_at = at * p.pieces + sub;
      scale_at = at * 2 * p.pieces + sub;
    }
  }
  const int n_pairs = (n_pieces + 1) / 2;
  const int k_lane = col * 64 + g * 16, v_lane = lane * 16;
  // keys of piece 2 pair + u, and values of both; what is not there is asked for at the cache's beginning and left out below
  q8_u4 kc[2][NB], vc[2][NB];
  q8_f4 ks[2], vs[2];
  auto at_piece = [&](int i, int at) { return i < n_pieces ? max(__builtin_amdgcn_readlane(at, i), 0) : 0; };
  auto ask_keys = [&](int pair, int u) {
    const uint8_t* at = p.kcodes + (size_t)at_piece(2 * pair + u, piece_at) * (NB * Q8_BYTES);
    ks[u] = *(const q8_f4*)(p.scales + (size_t)at_piece(2 * pair + u, scale_at) * Q8_PIECE + 4 * g);
#pragma unroll
    for (int j = 0; j < NB; j++) kc[u][j] = load_maybe_once<ONCE>((const q8_u4*)(at + j * Q8_BYTES + k_lane));
  };
  auto ask_values = [&](int pair) {
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const uint8_t* at = p.vcodes + (size_t)at_piece(2 * pair + u, piece_at) * (NB * Q8_BYTES);
      vs[u] = *(const q8_f4*)(p.scales + ((size_t)at_piece(2 * pair + u, scale_at) + p.pieces) * Q8_PIECE + 4 * g);
#pragma unroll
      for (int j = 0; j < NB; j++) vc[u][j] = load_maybe_once<ONCE>((const q8_u4*)(at + j * Q8_BYTES + v_lane));
    }
  };
  if (wave < n_pairs) {
    ask_keys(wave, 0);
    ask_keys(wave, 1);
    ask_values(wave);
  }

  // the queries: channels 64 j + 16 g .. + 15 of head col
#if ZSE_ACT_BF16
  q8_b8 qf[NB][2];
#else
  float qf[NB][16];
#endif
  {
    const act_t* row = p.q + (size_t)r * p.q_stride + (size_t)head * p.hd;
#pragma unroll
    for (int j = 0; j < NB; j++)
#pragma unroll
      for (int s = 0; s < 2; s++) {
        const int c0 = 64 * j + 16 * g + 8 * s;
        q8_a8 x;
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = from_f32<act_t>(0.f);
        if (col < heads) {
          if (p.q_whole) {
            if (c0 < p.hd) x = *(const q8_a8*)(row + c0);
          } else {
#pragma unroll
            for (int e = 0; e < 8; e++)
              if (c0 + e < p.hd) x[e] = row[c0 + e];
          }
        }
#if ZSE_ACT_BF16
        qf[j][s] = x;
#else
#pragma unroll
        for (int e = 0; e < 8; e++) qf[j][8 * s + e] = x[e];
#endif
      }
  }

  float m = -INFINITY, l = 0.f;
  q8_f4 o[NB * 4];
#pragma unroll
  for (int t = 0; t < NB * 4; t++) o[t] = q8_f4{0.f, 0.f, 0.f, 0.f};
  for (int pair = wave; pair < n_pairs; pair += 4) {
    // scores of head col: keys 16 (p0 + 2 pair + u) + 4 g + i
    float z[2][4];
#if !ZSE_ACT_BF16
    float val[2][4];                 // z by its factor: the exponent below is taken from these with one rounding
#endif
#pragma unroll
    for (int u = 0; u < 2; u++) {
      q8_f4 s = {0.f, 0.f, 0.f, 0.f};
#if !ZSE_ACT_BF16
      q8_f4 s2 = s;                                    // two chains of sums: shorter, and side by side
#endif
#pragma unroll
      for (int j = 0; j < NB; j++) {
#if ZSE_ACT_BF16
        s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q8_operand<FMT>(kc[u][j][0], kc[u][j][1]), qf[j][0], s, 0, 0, 0);
        s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q8_operand<FMT>(kc[u][j][2], kc[u][j][3]), qf[j][1], s, 0, 0, 0);
#else
#pragma unroll
        for (int w = 0; w < 4; w++) {
          float x[4];
          q8_floats<FMT>(kc[u][j][w], x);
#pragma unroll
          for (int e = 0; e < 4; e++) {
            q8_f4& sum = e & 1 ? s2 : s;
            sum = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], qf[j][4 * w + e], sum, 0, 0, 0);
          }
        }
#endif
      }
#if !ZSE_ACT_BF16
      s += s2;
#endif
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float dot = s[i] * ks[u][i];
        if constexpr (CAP) {
#if ZSE_ACT_BF16
          z[u][i] = p.c2 - 2.f * p.c2 * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(p.k2 * dot) + 1.f);
#else
          val[u][i] = tanhf(p.k2 * dot);
          z[u][i] = p.c2 * val[u][i];
#endif
        } else {
          z[u][i] = p.k1 * dot;
#if !ZSE_ACT_BF16
          val[u][i] = dot;
#endif
        }
      }
    }
    if (pair + 4 < n_pairs) {
      ask_keys(pair + 4, 0);
      ask_keys(pair + 4, 1);
    }
    // keys outside of [begin, end) and in pages that are not there
    const int key0 = (p0 + 2 * pair) * Q8_PIECE;
    const int at0 = __builtin_amdgcn_readlane(piece_at, 2 * pair);
    const int at1 = 2 * pair + 1 < n_pieces ? __builtin_amdgcn_readlane(piece_at, 2 * pair + 1) : -1;
    const bool whole = key0 >= begin && key0 + 2 * Q8_PIECE <= end && at0 >= 0 && at1 >= 0;
    if (!whole) {
#pragma unroll
      for (int u = 0; u < 2; u++) {
        unsigned mask = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int key = key0 + u * Q8_PIECE + 4 * g + i;
          const bool seen = key >= begin && key < end && (u ? at1 : at0) >= 0;
          mask |= seen ? 255u << (8 * i) : 0u;
          z[u][i] = seen ? z[u][i] : -INFINITY;
          vs[u][i] = seen ? vs[u][i] : 0.f;
        }
        // a code that is no number would meet a weight of zero
#pragma unroll
        for (int j = 0; j < NB; j++)
#pragma unroll
          for (int b = 0; b < 4; b++) vc[u][j][b] &= mask;
      }
    }
    float top = z[0][0];
#pragma unroll
    for (int i = 1; i < 8; i++) top = fmaxf(top, z[i / 4][i % 4]);
    const float m_new = fmaxf(m, wave_max16_32(top)), base = m_new == -INFINITY ? 0.f : m_new;
    if (__any(m_new != m)) {
      const float keep = __builtin_amdgcn_exp2f(m - base);
      l *= keep;
#pragma unroll
      for (int t = 0; t < NB * 4; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) o[t][i] *= keep;
      m = m_new;
    }
    float w[2][4];
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
#if ZSE_ACT_BF16
        const float e = __builtin_amdgcn_exp2f(z[u][i] - base);
#else
        // a rounding of z is |z| 2^-24 of its weight, as much as everything else together
        const float by = __fmaf_rn(val[u][i], CAP ? p.c2 : p.k1, -base) + val[u][i] * p.rest;
        const float e = z[u][i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(by);
#endif
        l += e;
        w[u][i] = e * vs[u][i];
      }
#if ZSE_ACT_BF16
    // A weight meets the values as two numbers, its rounded value and what the rounding left (16 bits of mantissa): with the first alone
    // the results are 1.5 times as far from 64 bits (2.6e-3 of them instead of 1.7e-3, which is their own rounding), and the products
    // are not what bounds the kernel.
    q8_b8 pb, rest;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      pb[e] = (__bf16)w[e / 4][e % 4];
      rest[e] = (__bf16)(w[e / 4][e % 4] - (float)pb[e]);
    }
#pragma unroll
    for (int j = 0; j < NB; j++)
#pragma unroll
      for (int b = 0; b < 4; b++) {
        const q8_b8 v = q8_operand<FMT>(vc[0][j][b], vc[1][j][b]);
        o[4 * j + b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, pb, o[4 * j + b], 0, 0, 0);
        o[4 * j + b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, rest, o[4 * j + b], 0, 0, 0);
      }
#else
#pragma unroll
    for (int u = 0; u < 2; u++)
#pragma unroll
      for (int j = 0; j < NB; j++)
#pragma unroll
        for (int b = 0; b < 4; b++) {
          float x[4];
          q8_floats<FMT>(vc[u][j][b], x);
#pragma unroll
          for (int i = 0; i < 4; i++) o[4 * j + b] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], w[u][i], o[4 * j + b], 0, 0, 0);
        }
#endif
    if (pair + 4 < n_pairs) ask_values(pair + 4);
  }
  l = wave_add16_32(l);

  // the four waves' results: [wave][head][channels, then maximum and sum]
  constexpr int ROW = NB * 64 + 4;
  if (col < heads) {
    float* mine = s_join + (wave * heads + col) * ROW;
#pragma unroll
    for (int t = 0; t < NB * 4; t++) *(q8_f4*)(mine + 16 * t + 4 * g) = o[t];
    if (g == 0) {
      mine[NB * 64] = m;
      mine[NB * 64 + 1] = l;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * NB * 64; i += 256) {
    const int h = i / (NB * 64), c = i % (NB * 64);
    float mw[4], most = -INFINITY, sum = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < 4; w++) most = fmaxf(most, mw[w] = s_join[(w * heads + h) * ROW + NB * 64]);
    const float base = most == -INFINITY ? 0.f : most;
#pragma unroll
    for (int w = 0; w < 4; w++) {
      const float f = __builtin_amdgcn_exp2f(mw[w] - base);
      sum += f * s_join[(w * heads + h) * ROW + NB * 64 + 1];
      x += f * s_join[(w * heads + h) * ROW + c];
    }
    const size_t hd_at = (size_t)r * p.nh + kvh * group + head0 + h;
    if (DIRECT) {
      if (c < p.hd) p.out[hd_at * p.hd + c] = from_f32<act_t>(sum == 0.f ? 0.f : x / sum);
    } else {
      const size_t part = hd_at * splits + split;
      p.part_o[part * (NB * 64) + c] = x;
      if (c == 0) {
        p.part_ml[part * 2] = most;
        p.part_ml[part * 2 + 1] = sum;
      }
    }
  }
#endif
}

// Joins the chunks' results of a (head, request): four channels a thread, the chunks dealt to as many groups of threads as there are.
// What the first round reads is asked for before the request's length is known (one wait for memory instead of three; what lies
// behind its chunks is never used).
template <int NB>
__global__ __launch_bounds__(256) void attention_q8_join_kernel(Q8Attention p, int splits) {
  constexpr int LANES = NB * 16, GROUPS = 256 / LANES, AHEAD = GROUPS > 8 ? 4 : 8;
  static_assert(AHEAD * GROUPS <= 64, "the first round's factors are one wave's lanes");
  __shared__ float s_o[GROUPS][NB * 64];
  const int head = blockIdx.x, r = blockIdx.y, lane = threadIdx.x & 63, group = min((int)threadIdx.x / LANES, GROUPS - 1), at = threadIdx.x % LANES;
  const size_t row = ((size_t)r * p.nh + head) * splits;
  const int ctx = min(p.ctx_len[r], p.max_ctx), first = p.window > 0 ? max(0, ctx - p.window) : 0;
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2* ml = (const f2*)p.part_ml + row;
  const f2 mine = ml[min(lane, splits - 1)];
  const float* part = p.part_o + row * (NB * 64) + at * 4;
  q8_f4 x[AHEAD];
#pragma unroll
  for (int e = 0; e < AHEAD; e++) x[e] = *(const q8_f4*)(part + (size_t)min(group + e * GROUPS, splits - 1) * (NB * 64));
  const int n = ctx > 0 ? ((ctx + p.chunk - 1) >> p.chunk_shift) - (first >> p.chunk_shift) : 0;
  float most = lane < n ? mine[0] : -INFINITY;
  for (int i = lane + 64; i < n; i += 64) most = fmaxf(most, ml[i][0]);
  most = wave_max_whole(most);
  const float base = most == -INFINITY ? 0.f : most;
  // lane i's factor of chunk i, and the sum of what the wave's lanes hold
  float f = lane < n ? exp2f(mine[0] - base) : 0.f;
  float l = lane < n ? f * mine[1] : 0.f;
  q8_f4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int e = 0; e < AHEAD; e++) {
    const int i = group + e * GROUPS;
    const float w = __shfl(f, i & 63);
    if (i < n) o += w * x[e];
  }
  for (int i0 = AHEAD * GROUPS; i0 < n; i0 += AHEAD * GROUPS) {
    float w[AHEAD];
#pragma unroll
    for (int e = 0; e < AHEAD; e++) {
      const int i = min(i0 + group + e * GROUPS, n - 1);
      w[e] = ml[i][0];
      x[e] = *(const q8_f4*)(part + (size_t)i * (NB * 64));
    }
#pragma unroll
    for (int e = 0; e < AHEAD; e++)
      if (i0 + group + e * GROUPS < n) o += exp2f(w[e] - base) * x[e];
  }
  for (int i = lane + 64; i < n; i += 64) l += exp2f(ml[i][0] - base) * ml[i][1];
  l = wave_sum_whole(l);
  if (threadIdx.x < LANES * GROUPS) *(q8_f4*)&s_o[group][at * 4] = o;
  __syncthreads();
  for (int c = threadIdx.x; c < p.hd; c += 256) {
    float y = 0.f;
#pragma unroll
    for (int w = 0; w < GROUPS; w++) y += s_o[w][c];
    p.out[((size_t)r * p.nh + head) * p.hd + c] = from_f32<act_t>(l == 0.f ? 0.f : y / l);
  }
}

// ---------------------------------------------------------------- entry points
static int q8_refuses(const char* who, const void* kcodes, const void* vcodes, const void* scales, int nkv, int hd, int bs,
                      int num_pages, int format) {
  const char* why = nullptr;
  if (nkv <= 0 || hd <= 0 || hd > 256) why = "1 to 256 channels of one key head or more";
  else if (bs <= 0 || bs % Q8_PIECE != 0 || num_pages <= 0) why = "pages of 16, 32, 48, ... tokens, one page or more";
  else if ((long long)nkv * bs * q8_blocks(hd) * Q8_BLOCK >= (1ll << 31)) why = "pages of less than 2 GiB";
  else if (format != 0 && format != 1) why = "format 0 (int8) or 1 (e4m3)";
  else if (!kcodes || !vcodes || !scales || ((uintptr_t)kcodes | (uintptr_t)vcodes | (uintptr_t)scales) % 16 != 0)
    why = "codes and scales at addresses that are multiples of 16";
  return why ? zk_fail((std::string(who) + ": a cache in 8 bits has " + why).c_str()) : 0;
}
#define Q8_REQUIRE_CACHE(who) \
  if (const int rc = q8_refuses(who, kcodes, vcodes, scales, nkv, hd, bs, num_pages, format)) return rc

// Bytes from the first to the last of ``rows`` rows of ``width`` values of the activations' type, ``ld`` apart.
static size_t q8_span(long long ld, long long width, long long rows) { return ((rows - 1) * ld + width) * sizeof(act_t); }
static bool q8_meet(const void* a, size_t a_bytes, const void* b, size_t b_bytes) {
  return (uintptr_t)a < (uintptr_t)b + b_bytes && (uintptr_t)b < (uintptr_t)a + a_bytes;
}

// Blocks of a launch.  Written: the heads of four rows are dealt to as many blocks as that gives (4,092 rows of 32 heads and 2 x 16 of
// 128 channels by 1,024, 2,048, 4,096 and 8,192 blocks 36.1, 33.9, 33.1 and 34.9 us; more work out the same angles).  Read back: waves that take
// pieces in turn (64 pages of 8 heads in a range of 64,512 pieces, one at a time, by 2,048, 4,096 and 8,192 blocks 8.0, 8.1 and 10.4 us:
// empty blocks cost as much as others; 147,000 pieces that are all there 56.9, 56.3 and 56.2).
#define Q8_WRITE_BLOCKS 4096
#define Q8_READ_BLOCKS 2048

// Calls ``go`` with what is only known at run time as a constant.
template <typename F>
static void q8_by_format(int format, F go) {
  if (format == 0) go(std::integral_constant<int, 0>());
  else go(std::integral_constant<int, 1>());
}
template <typename F>
static void q8_by_flag(bool flag, F go) {
  if (flag) go(std::true_type());
  else go(std::false_type());
}

// Keys of a partial result, by what a request's table can hold.  us by 256, 512 and 1,024 keys (16-bit rows, 8 heads over 4 of 256
// channels): one request of 4,000 keys 10.8, 12.8, 18.9; 64 of them 98.6, 93.7, 91.4; one of 16,000 15.6, 15.3, 20.8; eight of
// them 56.3, 49.8, 47.9; one of 60,000 45.1, 33.5, 28.3.  32-bit products take eight times as long for as many keys: by 128, 256
// and 512, 8 heads over 2 of 128, three requests of up to 700 keys 10.2, 12.9, 19.7; 8 over 4 of 256, one of 16,000 29.4, 25.1, 33.9.
#define Q8_WIDE 8192                  // tokens of a table from which chunks are longer
#define Q8_WIDER 32768
static int q8_chunk(long long table_tokens) {
#if ZSE_ACT_BF16
  return table_tokens < Q8_WIDE ? 256 : table_tokens < Q8_WIDER ? 512 : 1024;
#else
  return table_tokens < Q8_WIDE ? 128 : 256;
#endif
}

// Chunks that a request of up to max_ctx tokens may meet.
static int q8_splits(int max_ctx, int window, int chunk) {
  const int all = (int)std::max(1ll, ((long long)max_ctx + chunk - 1) / chunk);
  return window > 0 ? (int)std::min<long long>(all, ((long long)window + chunk - 2) / chunk + 1) : all;
}

extern "C" {

// Bytes of the codes of ``num_pages`` pages, keys or values (0: sizes that the cache does not take).
size_t zk_cache_q8_bytes(int num_pages, int nkv, int hd, int bs) {
  if (num_pages <= 0 || nkv <= 0 || hd <= 0 || hd > 256 || bs <= 0 || bs % Q8_PIECE != 0) return 0;
  return (size_t)num_pages * nkv * bs * q8_blocks(hd) * Q8_BLOCK;
}

// Rotates the queries and keys of T rows (query heads, key heads, value heads, ``ld`` values apart, or ``sums`` float planes
// [T][(nh + 2 nkv) hd] to add up, then rounded to the activations' type), stores the queries in rows of ``ldq`` values at q_out
// (qkv itself, where ldq is ld, is allowed; not the planes) and the keys and values in 8 bits at slot_map[t] = page * bs + offset.  A slot below
// zero or behind the last page is not stored; the slots of one call are distinct.  slot_map may be null, nkv zero: queries only.
int zk_rope_cache_write_q8(const void* qkv, int ld, const float* planes, int sums, void* q_out, int ldq, const int* positions,
                           const int* slot_map, const float* inv_freq, int rotary_dim, void* kcodes, void* vcodes, void* scales, int T,
                           int nh, int nkv, int hd, int bs, int num_pages, int format, void* stream) {
  ZK_REQUIRE(T >= 0 && nh > 0 && nkv >= 0 && sums >= 0, "zk_rope_cache_write_q8: bad sizes");
  ZK_REQUIRE(hd > 0 && hd <= 256, "zk_rope_cache_write_q8: heads of 1 to 256 channels");
  ZK_REQUIRE(nh <= 16384 && nkv <= 16384, "zk_rope_cache_write_q8: too many heads");
  if (nkv > 0 && slot_map) Q8_REQUIRE_CACHE("zk_rope_cache_write_q8");
  ZK_REQUIRE(nkv == 0 || !slot_map || (long long)num_pages * nkv * 2 * bs < (1ll << 31), "zk_rope_cache_write_q8: too many pages");
  ZK_REQUIRE(format == 0 || format == 1, "zk_rope_cache_write_q8: format 0 (int8) or 1 (e4m3)");
  ZK_REQUIRE(rotary_dim >= 0 && rotary_dim <= hd && rotary_dim % 2 == 0,
             "zk_rope_cache_write_q8: rotary_dim must be even and at most head_dim");
  ZK_REQUIRE(rotary_dim == 0 || inv_freq != nullptr, "zk_rope_cache_write_q8: no frequency table");
  ZK_REQUIRE(ldq >= nh * hd && (sums > 0 || ld >= (nh + 2 * nkv) * hd), "zk_rope_cache_write_q8: rows overlap");
  if (T == 0) return 0;
  ZK_REQUIRE(q_out && positions && (sums > 0 ? planes != nullptr && (uintptr_t)planes % 16 == 0 : qkv != nullptr),
             "zk_rope_cache_write_q8: null or misaligned argument");
  const int width = (nh + 2 * nkv) * hd, blocks = q8_blocks(hd);
  const bool partial = sums > 0;
  const size_t q_bytes = q8_span(ldq, (long long)nh * hd, T);
  ZK_REQUIRE(partial || (q_out == qkv && ldq == ld) || !q8_meet(qkv, q8_span(ld, width, T), q_out, q_bytes),
             "zk_rope_cache_write_q8: queries may go where they came from, in rows as far apart, or elsewhere");
  ZK_REQUIRE(!partial || !q8_meet(planes, (size_t)sums * T * width * sizeof(float), q_out, q_bytes),
             "zk_rope_cache_write_q8: queries over the partial sums");
  const int row = partial ? width : ld, heads = slot_map ? nh + 2 * nkv : nh;
  const bool whole = hd % 4 == 0 && rotary_dim % 8 == 0 && row % 4 == 0 && ldq % 4 == 0 && (uintptr_t)q_out % (4 * sizeof(act_t)) == 0 &&
                     (partial || (uintptr_t)qkv % (4 * sizeof(act_t)) == 0);
  const int lanes = blocks == 1 ? 16 : blocks == 2 ? 32 : 64, passes = (heads + 256 / lanes - 1) / (256 / lanes), groups = (T + 3) / 4;
  const dim3 grid(groups, std::max(1, std::min(passes, Q8_WRITE_BLOCKS / groups)));
  auto launch = [&](auto format_of, auto lanes_of, auto whole_of, auto partial_of) {
    constexpr bool SUMS = decltype(partial_of)::value;
    const Q8Write<SUMS> p{{(const act_t*)qkv, planes, row, sums, (size_t)T * width}, (act_t*)q_out, positions, slot_map, inv_freq,
                          (uint8_t*)kcodes, (uint8_t*)vcodes, (float*)scales, ldq, rotary_dim, T, nh, nkv, hd, bs, q8_shift(bs), num_pages, heads};
    write_q8_kernel<decltype(format_of)::value, decltype(lanes_of)::value, decltype(whole_of)::value, SUMS>
        <<<grid, 256, 0, (hipStream_t)stream>>>(p);
  };
  q8_by_format(format, [&](auto f) {
    q8_by_flag(whole, [&](auto w) {
      q8_by_flag(partial, [&](auto s) {
        if (lanes == 16) launch(f, std::integral_constant<int, 16>(), w, s);
        else if (lanes == 32) launch(f, std::integral_constant<int, 32>(), w, s);
        else launch(f, std::integral_constant<int, 64>(), w, s);
      });
    });
  });
  return zk_launch_status("zk_rope_cache_write_q8");
}

// Reads the pages back that requests 0 .. R-1 see, into the same pages of k and v [num_pages][nkv][bs][hd] in the activations' type
// (v_transposed: values as [num_pages][nkv][hd][bs]).  A request of ctx_len[r] tokens, the last q_start[r + 1] - q_start[r] of
// them new (q_start null: one), sees positions from max(0, ctx - new + 1 - window) on, all without a window.  Slots behind its last
// token are read as zeros; other pages stay as they were.  A page belongs to one request (one that two requests name is read as either
// of them sees it).
int zk_cache_read_q8(const void* kcodes, const void* vcodes, const float* scales, const int* block_table, int max_blocks,
                     const int* q_start, const int* ctx_len, void* k, void* v, int R, int max_ctx, int window, int nkv, int hd, int bs,
                     int num_pages, int v_transposed, int format, void* stream) {
  Q8_REQUIRE_CACHE("zk_cache_read_q8");
  ZK_REQUIRE(R >= 0 && max_ctx >= 0 && window >= 0 && max_blocks >= 0, "zk_cache_read_q8: bad sizes");
  ZK_REQUIRE(max_ctx <= 1 << 30, "zk_cache_read_q8: contexts of more than 2^30 tokens");
  ZK_REQUIRE(max_ctx <= (long long)max_blocks * bs, "zk_cache_read_q8: contexts longer than the table");
  ZK_REQUIRE(nkv <= 65535 && R <= 65535, "zk_cache_read_q8: too many requests or heads");
  if (R == 0 || max_ctx == 0) return 0;
  ZK_REQUIRE(block_table && ctx_len && k && v && ((uintptr_t)k | (uintptr_t)v) % 16 == 0, "zk_cache_read_q8: null or misaligned argument");
  if (window >= max_ctx) window = 0;                   // (sums of ctx, rows and window stay in 32 bits)
  Q8Read p;
  p.kcodes = (const uint8_t*)kcodes;
  p.vcodes = (const uint8_t*)vcodes;
  p.scales = scales;
  p.block_table = block_table;
  p.q_start = q_start;
  p.ctx_len = ctx_len;
  p.k = (act_t*)k;
  p.v = (act_t*)v;
  p.max_blocks = max_blocks;
  p.max_ctx = max_ctx;
  p.window = window;
  p.nkv = nkv;
  p.hd = hd;
  p.bs = bs;
  p.bs_shift = q8_shift(bs);
  p.num_pages = num_pages;
  p.R = R;
  // how much of it the requests' windows cover is not known here: blocks enough to fill the chip, whose waves take pieces in turn
  const long long pieces = ((max_ctx + (long long)bs - 1) / bs) * (bs / Q8_PIECE) * nkv * R;
  ZK_REQUIRE(pieces < (1ll << 30), "zk_cache_read_q8: too many pages");
  const int grid = (int)std::min<long long>((pieces + 3) / 4, Q8_READ_BLOCKS);
  // pairs where they make whole runs of 64 bytes (four windows of 4,096 in pages of 32, 8 heads of 256: 56.8 -> 54.8 us)
  auto launch = [&](auto f, auto t, auto w, auto u) {
    read_q8_kernel<decltype(f)::value, decltype(t)::value, decltype(w)::value, decltype(u)::value><<<grid, 256, 0, (hipStream_t)stream>>>(p);
  };
  q8_by_format(format, [&](auto f) {
    q8_by_flag(hd % 8 == 0, [&](auto w) {
      if (!v_transposed) launch(f, std::false_type(), w, std::false_type());
#if ZSE_ACT_BF16
      else if (bs % (2 * Q8_PIECE) == 0) launch(f, std::true_type(), w, std::true_type());
#endif
      else launch(f, std::true_type(), w, std::false_type());
    });
  });
  return zk_launch_status("zk_cache_read_q8");
}

// Bytes of workspace of zk_attention_q8 for up to R requests of up to max_ctx tokens in tables that reach up to table_tokens: what is
// enough for the largest of each is enough for less.  (A narrower table may need more: its chunks are shorter.)
size_t zk_attention_q8_workspace(int R, int nh, int hd, int max_ctx, int table_tokens) {
  if (R <= 0 || nh <= 0 || hd <= 0 || hd > 256 || max_ctx <= 0) return 0;
  const int widest = std::max(max_ctx, table_tokens);
  int splits = q8_splits(max_ctx, 0, q8_chunk(widest));
  for (const int narrower : {Q8_WIDE - 1, Q8_WIDER - 1})         // the widest of shorter chunks
    if (narrower < widest) splits = std::max(splits, q8_splits(std::min(max_ctx, narrower), 0, q8_chunk(narrower)));
  return (size_t)R * nh * splits * (q8_blocks(hd) * Q8_BLOCK + 2) * sizeof(float);
}

// Attention of one token a request, the last of its ctx_len[r], over its cache: z_j = scale q.k_j (softcap > 0: softcap
// tanh(z_j / softcap)) for j from max(0, ctx - window) on (all without a window), out = sum softmax(z)_j v_j.  In 16 bits a capped
// score is off by up to softcap 2^-20: caps are tens, not hundred thousands.  q: row r at r * q_stride;
// out: rows of nh * hd, apart from q.  A request without keys gets zeros, and a page that the table does not name (below zero, or not below
// num_pages) has none.
int zk_attention_q8(const void* q, int q_stride, const void* kcodes, const void* vcodes, const float* scales, const int* block_table,
                    int max_blocks, const int* ctx_len, void* out, int R, int max_ctx, int nh, int nkv, int hd, int bs, int num_pages,
                    float scale, float softcap, int window, int format, void* workspace, size_t workspace_bytes, void* stream) {
  Q8_REQUIRE_CACHE("zk_attention_q8");
  ZK_REQUIRE(R >= 0 && max_ctx >= 0 && window >= 0 && max_blocks >= 0 && nh > 0, "zk_attention_q8: bad sizes");
  ZK_REQUIRE(nh % nkv == 0, "zk_attention_q8: query heads must be a multiple of key heads");
  ZK_REQUIRE(nh <= 65535 && R <= 65535, "zk_attention_q8: too many heads or requests");
  ZK_REQUIRE(q_stride >= (long long)nh * hd, "zk_attention_q8: rows overlap");
  ZK_REQUIRE(max_ctx <= 1 << 30, "zk_attention_q8: contexts of more than 2^30 tokens");
  ZK_REQUIRE(max_ctx <= (long long)max_blocks * bs, "zk_attention_q8: contexts longer than the table");
  ZK_REQUIRE((long long)num_pages * nkv * 2 * (bs / Q8_PIECE) < (1ll << 31), "zk_attention_q8: too many pages");
  ZK_REQUIRE(softcap >= 0.f && softcap <= FLT_MAX, "zk_attention_q8: softcap must be finite and not negative (0: no cap)");
  if (R == 0) return 0;
  ZK_REQUIRE(q && out && ctx_len && (block_table || max_ctx == 0), "zk_attention_q8: null argument");
  ZK_REQUIRE(!q8_meet(q, q8_span(q_stride, (long long)nh * hd, R), out, (size_t)R * nh * hd * sizeof(act_t)), "zk_attention_q8: results over queries");
  if (window >= max_ctx) window = 0;                   // (sums of ctx and window stay in 32 bits)
  Q8Attention p;
  p.chunk = q8_chunk((long long)max_blocks * bs);
  const int splits = q8_splits(max_ctx, window, p.chunk), blocks = q8_blocks(hd);
  const size_t row = (size_t)R * nh * splits;
  ZK_REQUIRE(splits <= 65535, "zk_attention_q8: contexts of too many chunks");
  if (splits > 1) {
    ZK_REQUIRE(workspace && (uintptr_t)workspace % 16 == 0, "zk_attention_q8: no workspace, or not at a multiple of 16");
    ZK_REQUIRE(workspace_bytes >= row * (blocks * Q8_BLOCK + 2) * sizeof(float), "zk_attention_q8: the workspace is too small");
  }
  p.q = (const act_t*)q;
  p.kcodes = (const uint8_t*)kcodes;
  p.vcodes = (const uint8_t*)vcodes;
  p.scales = scales;
  p.block_table = block_table;
  p.ctx_len = ctx_len;
  p.out = (act_t*)out;
  p.part_o = (float*)workspace;
  p.part_ml = splits > 1 ? (float*)workspace + row * blocks * Q8_BLOCK : nullptr;
  p.q_stride = q_stride;
  p.max_blocks = max_blocks;
  p.max_ctx = max_ctx;
  p.nh = nh;
  p.nkv = nkv;
  p.hd = hd;
  p.pieces = bs / Q8_PIECE;
  p.pieces_shift = q8_shift(p.pieces);
  p.chunk_shift = q8_shift(p.chunk);
  p.num_pages = num_pages;
  p.window = window;
  // queries by loads of eight, where heads and rows are whole such pieces
  p.q_whole = hd % 8 == 0 && q_stride % 8 == 0 && (uintptr_t)q % (8 * sizeof(act_t)) == 0;
  const double log2e = 1.4426950408889634;
  p.k1 = (float)(scale * log2e);
#if ZSE_ACT_BF16
  p.k2 = softcap > 0.f ? (float)(2.0 * scale / softcap * log2e) : 0.f;
#else
  p.k2 = softcap > 0.f ? scale / softcap : 0.f;
#endif
  p.c2 = (float)(softcap * log2e);
  p.rest = softcap > 0.f ? (float)(softcap * log2e - p.c2) : (float)(scale * log2e - p.k1);
  const int group = nh / nkv, tiles = (group + 15) / 16;
  const dim3 grid(nkv * tiles, R, splits);
  // Codes past the caches where one block alone reads them and R requests of max_ctx keys are more than the memory side's cache holds.  A
  // window is not taken off: what it leaves of a layer may fit, what all layers of a step read does not (behind a window of 4,096, one layer
  // over and over / eight in turn: 8 requests of 20,000, 4 heads of 256, 20.9 / 22.5 us past the caches, 20.3 / 24.1 through them; 4 of 60,000, 8
  // heads of 128, 17.6 / 19.2 and 16.9 / 19.1).
  const bool once = tiles == 1 && (double)R * max_ctx * nkv * (2 * blocks * Q8_BLOCK + 8) > 256.0 * (1 << 20);
  const size_t lds = (size_t)4 * std::min(group, 16) * (blocks * Q8_BLOCK + 4) * sizeof(float);
#define Q8_KERNEL(FMT, NB, CAP, DIRECT) (once ? attention_q8_kernel<FMT, NB, CAP, DIRECT, true> : attention_q8_kernel<FMT, NB, CAP, DIRECT, false>)
#define Q8_ATTEND(FMT, NB)                                                                                             \
  do {                                                                                                                 \
    const auto kernel = softcap > 0.f ? (splits > 1 ? Q8_KERNEL(FMT, NB, true, false) : Q8_KERNEL(FMT, NB, true, true))    \
                                      : (splits > 1 ? Q8_KERNEL(FMT, NB, false, false) : Q8_KERNEL(FMT, NB, false, true)); \
    if (lds > (64 << 10)) {                                                                                            \
      const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds); \
      if (e != hipSuccess) return zk_fail("zk_attention_q8: no room in LDS");                                          \
    }                                                                                                                  \
    kernel<<<grid, 256, lds, (hipStream_t)stream>>>(p);                                                                \
    if (splits > 1) attention_q8_join_kernel<NB><<<dim3(nh, R), 256, 0, (hipStream_t)stream>>>(p, splits);             \
  } while (0)
#define Q8_BY_BLOCKS(FMT)                    \
  switch (blocks) {                          \
    case 1: Q8_ATTEND(FMT, 1); break;        \
    case 2: Q8_ATTEND(FMT, 2); break;        \
    case 3: Q8_ATTEND(FMT, 3); break;        \
    default: Q8_ATTEND(FMT, 4); break;       \
  }
  if (format == 0) {
    Q8_BY_BLOCKS(0)
  } else {
    Q8_BY_BLOCKS(1)
  }
#undef Q8_BY_BLOCKS
#undef Q8_ATTEND
#undef Q8_KERNEL
  return zk_launch_status("zk_attention_q8");
}

}  // extern "C"

ZK_ENTER(zk_rope_cache_write_q8)
ZK_ENTER(zk_cache_read_q8)
ZK_ENTER(zk_attention_q8)
