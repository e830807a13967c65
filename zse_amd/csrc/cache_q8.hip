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

#include <cfloat>

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

template <int FMT>
__device__ __forceinline__ float q8_top() { return FMT == 0 ? 127.f : 448.f; }
template <int FMT>
__device__ __forceinline__ unsigned q8_code(float x) {          // of a value times top / a
  if constexpr (FMT == 0) return (unsigned)(int)fminf(fmaxf(rintf(x), -127.f), 127.f) & 255u;
  else {
    x = fminf(fmaxf(x, -448.f), 448.f);
#ifdef __HIP_DEVICE_COMPILE__
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(x, x, 0, false) & 255u;
#else
    return 0;
#endif
  }
}
template <int FMT>
__device__ __forceinline__ float q8_number(unsigned code) {
  if constexpr (FMT == 0) return (float)(int)(int8_t)code;
  else {
#ifdef __HIP_DEVICE_COMPILE__
    return __builtin_amdgcn_cvt_f32_fp8((int)code, 0);
#else
    return 0.f;
#endif
  }
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
    scale = __fdiv_rn(a, top);
    factor = __fdiv_rn(top, a);
  }
}
// A value times its factor; 0 in a head whose scale says that nothing can be held.
__device__ __forceinline__ float q8_times(float x, float factor) { return factor == 0.f ? 0.f : __fmul_rn(x, factor); }

// The larger of two magnitudes, NaN if one is.
__device__ __forceinline__ float q8_larger(float a, float b) { return a != a || b != b ? __int_as_float(0x7fc00000) : fmaxf(a, b); }

// Sine and cosine of pos * freq, positions below 2^24.  The product is held in two floats (rounded to one it is off by up to half
// a step of the angle, 2^-12 at position 4,096 and 2^-7 at 131,072), less whole turns (2 pi in two floats; n times the first
// takes nothing from a multiple of its last place), then one float and what that leaves, which turns the result to first order.
__device__ __forceinline__ void q8_sincos(float pos, float freq, float& sn, float& cs) {
  const float angle = __fmul_rn(pos, freq), low = __fmaf_rn(pos, freq, -angle);
  const float n = rintf(angle * 0.15915494f);
  const float a = __fmaf_rn(n, -6.2831855f, angle), b = __fmaf_rn(n, 1.7484556e-7f, low);
  const float r = a + b, part = r - a, rest = (a - (r - part)) + (b - part);
  float s, c;
  sincosf(r, &s, &c);
  sn = __fmaf_rn(c, rest, s);
  cs = __fmaf_rn(s, -rest, c);
}

// ---------------------------------------------------------------- written
struct Q8Rows {
  const act_t* rows;
  const float* planes;        // partial sums of a split product, or none
  int ld, sums;
  size_t plane;
  __device__ __forceinline__ float at(size_t t, int i) const {
    if (sums <= 0) return to_f32(rows[t * ld + i]);
    float x = planes[t * ld + i];
    for (int p = 1; p < sums; p++) x += planes[p * plane + t * ld + i];
    return to_f32(from_f32<act_t>(x));
  }
};

template <int FMT>
__global__ __launch_bounds__(64) void write_q8_kernel(Q8Rows from, act_t* q_out, int ldq, const int* __restrict__ positions,
                                                      const int* __restrict__ slot_map, const float* __restrict__ inv_freq, int rotary_dim,
                                                      uint8_t* __restrict__ kcodes, uint8_t* __restrict__ vcodes, float* __restrict__ scales,
                                                      int nh, int nkv, int hd, int bs, int num_pages) {
  const int t = blockIdx.x, head = blockIdx.y, lane = threadIdx.x, half = rotary_dim / 2;
  const bool is_q = head < nh, is_v = head >= nh + nkv;
  const int slot = slot_map && !is_q ? slot_map[t] : -1;
  const bool store = slot >= 0 && slot / bs < num_pages;
  if (!is_q && !store) return;
  const float pos = (float)positions[t];
  float x[4];
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const int c = lane + 64 * e;
    x[e] = 0.f;
    if (c >= hd) continue;
    x[e] = from.at(t, head * hd + c);
    if (!is_v && c < rotary_dim) {
      const int i = c < half ? c : c - half;
      const float other = from.at(t, head * hd + (c < half ? c + half : i));
      float sn, cs, ra, rb;
      q8_sincos(pos, inv_freq[i], sn, cs);
      rotate_pair(c < half ? x[e] : other, c < half ? other : x[e], sn, cs, ra, rb);
      x[e] = c < half ? ra : rb;
    }
  }
  if (is_q) {
#pragma unroll
    for (int e = 0; e < 4; e++)
      if (lane + 64 * e < hd) q_out[(size_t)t * ldq + head * hd + lane + 64 * e] = from_f32<act_t>(x[e]);
    return;
  }
  float a = 0.f;
#pragma unroll
  for (int e = 0; e < 4; e++) a = q8_larger(a, fabsf(x[e]));
  const float bad = wave_max_whole(a != a ? 1.f : 0.f);
  a = bad > 0.f ? __int_as_float(0x7fc00000) : wave_max_whole(a);
  float scale, factor;
  q8_scales<FMT>(a, scale, factor);
  const int kvh = (head - nh) % nkv, page = slot / bs, off = slot % bs, blocks = q8_blocks(hd);
  uint8_t* dst = (is_v ? vcodes : kcodes) + q8_piece(page, off / Q8_PIECE, kvh, nkv, bs / Q8_PIECE, blocks);
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (e < blocks)
      dst[e * Q8_BYTES + (is_v ? q8_value_at(off % Q8_PIECE, lane) : q8_key_at(off % Q8_PIECE, lane))] =
          (uint8_t)q8_code<FMT>(q8_times(x[e], factor));
  if (lane == 0) scales[q8_scale(page, kvh, nkv, bs, is_v) + off] = scale;
}

// ---------------------------------------------------------------- read back
template <int FMT>
__global__ __launch_bounds__(256) void read_q8_kernel(const uint8_t* __restrict__ kcodes, const uint8_t* __restrict__ vcodes,
                                                      const float* __restrict__ scales, const int* __restrict__ block_table, int max_blocks,
                                                      const int* __restrict__ q_start, const int* __restrict__ ctx_len, act_t* __restrict__ k,
                                                      act_t* __restrict__ v, int max_ctx, int window, int nkv, int hd, int bs, int num_pages,
                                                      int v_transposed) {
  const int j = blockIdx.x, head = blockIdx.y, r = blockIdx.z;
  const int ctx = min(ctx_len[r], max_ctx);
  const int rows = q_start ? q_start[r + 1] - q_start[r] : 1;
  const int first = window > 0 ? max(0, ctx - rows + 1 - window) : 0;
  if (j < first / bs || j * bs >= ctx) return;
  const int page = block_table[(size_t)r * max_blocks + j];
  if (page < 0 || page >= num_pages) return;
  const int there = min(bs, ctx - j * bs), blocks = q8_blocks(hd);
  const size_t out = ((size_t)page * nkv + head) * (size_t)(bs * hd);
  for (int i = threadIdx.x; i < bs * hd; i += 256) {
    const int t = i / hd, c = i % hd;
    const size_t at = q8_piece(page, t / Q8_PIECE, head, nkv, bs / Q8_PIECE, blocks) + c / Q8_BLOCK * Q8_BYTES;
    float x = 0.f, y = 0.f;
    if (t < there) {
      x = q8_number<FMT>(kcodes[at + q8_key_at(t % Q8_PIECE, c % Q8_BLOCK)]) * scales[q8_scale(page, head, nkv, bs, 0) + t];
      y = q8_number<FMT>(vcodes[at + q8_value_at(t % Q8_PIECE, c % Q8_BLOCK)]) * scales[q8_scale(page, head, nkv, bs, 1) + t];
    }
    k[out + i] = from_f32<act_t>(x);
    v[out + (v_transposed ? c * bs + t : i)] = from_f32<act_t>(y);
  }
}

// ---------------------------------------------------------------- attended to
// One wave a (request, head): 64 keys at a time, a lane a key for the scores, lanes over the channels for the values.
template <int FMT>
__global__ __launch_bounds__(64) void attention_q8_kernel(const act_t* __restrict__ q, int q_stride, const uint8_t* __restrict__ kcodes,
                                                          const uint8_t* __restrict__ vcodes, const float* __restrict__ scales,
                                                          const int* __restrict__ block_table, int max_blocks,
                                                          const int* __restrict__ ctx_len, act_t* __restrict__ out, int max_ctx, int nh,
                                                          int nkv, int hd, int bs, int num_pages, float scale, float softcap, int window) {
  __shared__ float s_p[64];
  __shared__ size_t s_at[64];
  __shared__ int s_page[64];
  const int r = blockIdx.x, head = blockIdx.y, lane = threadIdx.x, kvh = head / (nh / nkv), blocks = q8_blocks(hd), pieces = bs / Q8_PIECE;
  const int ctx = min(ctx_len[r], max_ctx), first = window > 0 ? max(0, ctx - window) : 0;
  const act_t* row = q + (size_t)r * q_stride + (size_t)head * hd;
  float m = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int j0 = first; j0 < ctx; j0 += 64) {
    const int j = j0 + lane;
    const int page = j < ctx ? block_table[(size_t)r * max_blocks + j / bs] : -1;
    float z = -INFINITY, vs = 0.f;
    size_t at = 0;
    const bool seen = page >= 0 && page < num_pages;
    if (seen) {
      const int off = j % bs;
      at = q8_piece(page, off / Q8_PIECE, kvh, nkv, pieces, blocks);
      float dot = 0.f;
      for (int c = 0; c < hd; c++)
        dot += to_f32(row[c]) * q8_number<FMT>(kcodes[at + c / 64 * Q8_BYTES + q8_key_at(off % Q8_PIECE, c % 64)]);
      z = dot * scales[q8_scale(page, kvh, nkv, bs, 0) + off] * scale;
      if (softcap > 0.f) z = softcap * tanhf(z / softcap);
      vs = scales[q8_scale(page, kvh, nkv, bs, 1) + off];
    }
    const float bad = wave_max_whole(seen && z != z ? 1.f : 0.f);
    const float now = fmaxf(m, wave_max_whole(z)), base = now == -INFINITY ? 0.f : now;
    const float keep = expf(m - base);
    float p = seen ? expf(z - base) : 0.f;
    if (bad > 0.f) p = __int_as_float(0x7fc00000);
    l = l * keep + wave_sum_whole(p);
    m = now;
    __syncthreads();
    s_p[lane] = seen ? p * vs : 0.f;
    s_at[lane] = at;
    s_page[lane] = seen ? j % bs % Q8_PIECE : -1;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 4; e++) {
      if (lane + 64 * e >= hd) continue;
      float sum = 0.f;
      for (int i = 0; i < 64; i++)
        if (s_page[i] >= 0) sum += s_p[i] * q8_number<FMT>(vcodes[s_at[i] + e * Q8_BYTES + q8_value_at(s_page[i], lane)]);
      acc[e] = acc[e] * keep + sum;
    }
  }
#pragma unroll
  for (int e = 0; e < 4; e++)
    if (lane + 64 * e < hd) out[((size_t)r * nh + head) * hd + lane + 64 * e] = from_f32<act_t>(l == 0.f ? 0.f : acc[e] / l);
}

// ---------------------------------------------------------------- entry points
static int q8_refuses(const char* who, const void* kcodes, const void* vcodes, const void* scales, int nkv, int hd, int bs,
                      int num_pages, int format) {
  const char* why = nullptr;
  if (nkv <= 0 || hd <= 0 || hd > 256) why = "1 to 256 channels of one key head or more";
  else if (bs <= 0 || bs % Q8_PIECE != 0 || num_pages <= 0) why = "pages of 16, 32, 48, ... tokens, one page or more";
  else if (format != 0 && format != 1) why = "format 0 (int8) or 1 (e4m3)";
  else if (!kcodes || !vcodes || !scales || ((uintptr_t)kcodes | (uintptr_t)vcodes | (uintptr_t)scales) % 16 != 0)
    why = "codes and scales at addresses that are multiples of 16";
  return why ? zk_fail((std::string(who) + ": a cache in 8 bits has " + why).c_str()) : 0;
}
#define Q8_REQUIRE_CACHE(who) \
  if (const int rc = q8_refuses(who, kcodes, vcodes, scales, nkv, hd, bs, num_pages, format)) return rc
#define Q8_FORMAT(call)            \
  if (format == 0) {               \
    constexpr int FMT = 0;         \
    call;                          \
  } else {                         \
    constexpr int FMT = 1;         \
    call;                          \
  }

extern "C" {

// Bytes of the codes of ``num_pages`` pages, keys or values (0: sizes that the cache does not take).
size_t zk_cache_q8_bytes(int num_pages, int nkv, int hd, int bs) {
  if (num_pages <= 0 || nkv <= 0 || hd <= 0 || hd > 256 || bs <= 0 || bs % Q8_PIECE != 0) return 0;
  return (size_t)num_pages * nkv * bs * q8_blocks(hd) * Q8_BLOCK;
}

// Rotates the queries and keys of T rows (query heads, key heads, value heads, ``ld`` values apart, or ``sums`` float planes
// [T][(nh + 2 nkv) hd] to add up, then rounded to the activations' type), stores the queries in rows of ``ldq`` values at q_out
// (qkv itself, where ldq is ld, is allowed) and the keys and values in 8 bits at slot_map[t] = page * bs + offset.  A slot below
// zero or behind the last page is not stored; the slots of one call are distinct.  slot_map may be null, nkv zero: queries only.
int zk_rope_cache_write_q8(const void* qkv, int ld, const float* planes, int sums, void* q_out, int ldq, const int* positions,
                           const int* slot_map, const float* inv_freq, int rotary_dim, void* kcodes, void* vcodes, void* scales, int T,
                           int nh, int nkv, int hd, int bs, int num_pages, int format, void* stream) {
  ZK_REQUIRE(T >= 0 && nh > 0 && nkv >= 0 && sums >= 0, "zk_rope_cache_write_q8: bad sizes");
  ZK_REQUIRE(hd > 0 && hd <= 256, "zk_rope_cache_write_q8: heads of 1 to 256 channels");
  ZK_REQUIRE(nh <= 16384 && nkv <= 16384, "zk_rope_cache_write_q8: too many heads");
  if (nkv > 0 && slot_map) Q8_REQUIRE_CACHE("zk_rope_cache_write_q8");
  ZK_REQUIRE(format == 0 || format == 1, "zk_rope_cache_write_q8: format 0 (int8) or 1 (e4m3)");
  ZK_REQUIRE(rotary_dim >= 0 && rotary_dim <= hd && rotary_dim % 2 == 0,
             "zk_rope_cache_write_q8: rotary_dim must be even and at most head_dim");
  ZK_REQUIRE(rotary_dim == 0 || inv_freq != nullptr, "zk_rope_cache_write_q8: no frequency table");
  ZK_REQUIRE(ldq >= nh * hd && (sums > 0 || ld >= (nh + 2 * nkv) * hd), "zk_rope_cache_write_q8: rows overlap");
  if (T == 0) return 0;
  ZK_REQUIRE(q_out && positions && (sums > 0 ? planes != nullptr && (uintptr_t)planes % 16 == 0 : qkv != nullptr),
             "zk_rope_cache_write_q8: null or misaligned argument");
  const int width = (nh + 2 * nkv) * hd;
  const Q8Rows from{(const act_t*)qkv, planes, sums > 0 ? width : ld, sums, (size_t)T * width};
  Q8_FORMAT((write_q8_kernel<FMT><<<dim3(T, slot_map ? nh + 2 * nkv : nh), 64, 0, (hipStream_t)stream>>>(
      from, (act_t*)q_out, ldq, positions, slot_map, inv_freq, rotary_dim, (uint8_t*)kcodes, (uint8_t*)vcodes, (float*)scales, nh, nkv, hd,
      bs, num_pages)))
  return zk_launch_status("zk_rope_cache_write_q8");
}

// Reads the pages back that requests 0 .. R-1 see, into the same pages of k and v [num_pages][nkv][bs][hd] in the activations' type
// (v_transposed: values as [num_pages][nkv][hd][bs]).  A request of ctx_len[r] tokens, the last q_start[r + 1] - q_start[r] of
// them new (q_start null: one), sees positions from max(0, ctx - new + 1 - window) on, all without a window.  Slots behind its last
// token are read as zeros; other pages stay as they were.
int zk_cache_read_q8(const void* kcodes, const void* vcodes, const float* scales, const int* block_table, int max_blocks,
                     const int* q_start, const int* ctx_len, void* k, void* v, int R, int max_ctx, int window, int nkv, int hd, int bs,
                     int num_pages, int v_transposed, int format, void* stream) {
  Q8_REQUIRE_CACHE("zk_cache_read_q8");
  ZK_REQUIRE(R >= 0 && max_ctx >= 0 && window >= 0 && max_blocks >= 0, "zk_cache_read_q8: bad sizes");
  ZK_REQUIRE(max_ctx <= (long long)max_blocks * bs, "zk_cache_read_q8: contexts longer than the table");
  ZK_REQUIRE(nkv <= 65535 && R <= 65535, "zk_cache_read_q8: too many requests or heads");
  if (R == 0 || max_ctx == 0) return 0;
  ZK_REQUIRE(block_table && ctx_len && k && v && ((uintptr_t)k | (uintptr_t)v) % 16 == 0, "zk_cache_read_q8: null or misaligned argument");
  Q8_FORMAT((read_q8_kernel<FMT><<<dim3((max_ctx + bs - 1) / bs, nkv, R), 256, 0, (hipStream_t)stream>>>(
      (const uint8_t*)kcodes, (const uint8_t*)vcodes, scales, block_table, max_blocks, q_start, ctx_len, (act_t*)k, (act_t*)v, max_ctx,
      window, nkv, hd, bs, num_pages, v_transposed)))
  return zk_launch_status("zk_cache_read_q8");
}

// Bytes of workspace of zk_attention_q8 for R requests of up to max_ctx tokens whose table reaches table_tokens.
size_t zk_attention_q8_workspace(int R, int nh, int hd, int max_ctx, int table_tokens) { return 0; }

// Attention of one token a request, the last of its ctx_len[r], over its cache: z_j = scale q.k_j (softcap > 0: softcap
// tanh(z_j / softcap)) for j from max(0, ctx - window) on (all without a window), out = sum softmax(z)_j v_j.  q: row r at r * q_stride;
// out: rows of nh * hd.  A request without keys gets zeros, and a page that the table does not name (below zero, or not below
// num_pages) has none.
int zk_attention_q8(const void* q, int q_stride, const void* kcodes, const void* vcodes, const float* scales, const int* block_table,
                    int max_blocks, const int* ctx_len, void* out, int R, int max_ctx, int nh, int nkv, int hd, int bs, int num_pages,
                    float scale, float softcap, int window, int format, void* workspace, size_t workspace_bytes, void* stream) {
  Q8_REQUIRE_CACHE("zk_attention_q8");
  ZK_REQUIRE(R >= 0 && max_ctx >= 0 && window >= 0 && max_blocks >= 0 && nh > 0, "zk_attention_q8: bad sizes");
  ZK_REQUIRE(nh % nkv == 0, "zk_attention_q8: query heads must be a multiple of key heads");
  ZK_REQUIRE(nh <= 65535 && q_stride >= nh * hd, "zk_attention_q8: rows overlap, or too many heads");
  ZK_REQUIRE(max_ctx <= (long long)max_blocks * bs, "zk_attention_q8: contexts longer than the table");
  ZK_REQUIRE(softcap >= 0.f, "zk_attention_q8: softcap must not be negative");
  if (R == 0) return 0;
  ZK_REQUIRE(q && out && ctx_len && (block_table || max_ctx == 0), "zk_attention_q8: null argument");
  Q8_FORMAT((attention_q8_kernel<FMT><<<dim3(R, nh), 64, 0, (hipStream_t)stream>>>(
      (const act_t*)q, q_stride, (const uint8_t*)kcodes, (const uint8_t*)vcodes, scales, block_table, max_blocks, ctx_len, (act_t*)out,
      max_ctx, nh, nkv, hd, bs, num_pages, scale, softcap, window)))
  return zk_launch_status("zk_attention_q8");
}

}  // extern "C"

ZK_ENTER(zk_rope_cache_write_q8)
ZK_ENTER(zk_cache_read_q8)
ZK_ENTER(zk_attention_q8)
