// The step in front of attention over ordinary key and value heads, in one pass over the projection's result: RMSNorm of every query
// and key head, rotary positions, and the new keys and values into their paged caches.
//
//   y = x * rsqrt(mean_d(x^2) + eps) * gamma                                      (where there is a gamma)
//   half pairs:        (y_i, y_{i+R/2}) -> (y_i c_i - y_{i+R/2} s_i, y_{i+R/2} c_i + y_i s_i),   i < R/2, R <= D
//   interleaved pairs: (y_2i, y_2i+1)   -> the same with the neighbour
//   c_i, s_i = the tables' entries of the token's position; elements from R on stay as they are
// in fp32 from the 16-bit inputs, rounded once: to the inputs' type, or for an 8-bit cache x / scale[head] to e4m3 (values beyond
// +-448 become +-448, NaN stays NaN).
//
// A group of 8, 16 or 32 lanes holds a head, eight values a lane; the norm's sum and a half pair's other element come by lane moves.
// A group takes several heads of one token, so that the token's table entries are read once (a lane's entries are four times its
// values' bytes).  What bounds it is memory: every value is read and written once.
#include "cache_rows.hpp"

namespace mlahip {
namespace heads {

struct PrologueParams {
  const char* src[3]; int64_t src_st[3], src_sh[3];          // q, k, v [T, heads, D]; strides in bytes
  char* out[2]; int64_t out_st[2], out_sh[2];                // rotated q, k as tensors (or null)
  char* cache[2]; int64_t c_sp[2], c_sr[2], c_sh[2];         // K and V cache [pages, page, heads, D], strides in bytes (or null)
  const char* gamma[2];
  const float* scale[2];                                     // of an 8-bit cache, a number per head (null: 1)
  const char *cos, *sin; int64_t cs_st; int64_t table_rows;  // bytes between positions
  const int64_t *positions, *slots;
  int64_t num_tokens, num_pages;
  int32_t page_size, q_heads, kv_heads, dim, rotary, table_f32;
  int32_t parts;                                             // groups that share a token's heads
  float eps;
};

template <typename T> struct Vec8 { typedef T type __attribute__((ext_vector_type(8))); };

// eight entries of a table from entry i on
__device__ __forceinline__ void entries(const char* row, int i, bool f32, float* e) {
  if (f32) {
    const f32x4 a = *(const f32x4*)(row + i * 4), b = *(const f32x4*)(row + i * 4 + 16);
#pragma unroll
    for (int j = 0; j < 4; j++) { e[j] = a[j]; e[4 + j] = b[j]; }
  } else {
    const bf16x8 a = *(const bf16x8*)(row + i * 2);
#pragma unroll
    for (int j = 0; j < 8; j++) e[j] = (float)a[j];
  }
}
__device__ __forceinline__ void entries4(const char* row, int i, bool f32, float* e) {
  if (f32) {
    const f32x4 a = *(const f32x4*)(row + i * 4);
#pragma unroll
    for (int j = 0; j < 4; j++) e[j] = a[j];
  } else {
    const bf16x4 a = *(const bf16x4*)(row + i * 2);
#pragma unroll
    for (int j = 0; j < 4; j++) e[j] = (float)a[j];
  }
}

// x / s to e4m3, saturated: the quotient by the reciprocal and one correction by the remainder (a division is ten instructions a value)
__device__ __forceinline__ u32x2 to_e4m3(const float* x, float s) {
  const float inv = 1.f / s;
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; e++) {
    float v = x[e] * inv;
    const float r = __builtin_fmaf(-v, s, x[e]);
    const float w = __builtin_fmaf(r, inv, v);
    v = __builtin_isfinite(v) ? w : v;
    y[e] = v != v ? v : fminf(fmaxf(v, -448.f), 448.f);
  }
  int w0 = 0, w1 = 0;
  w0 = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], w0, false);
  w0 = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w0, true);
  w1 = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], w1, false);
  w1 = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], w1, true);
  return u32x2{(uint32_t)w0, (uint32_t)w1};
}

// T: the inputs' type; kLanes: lanes of a head; kFp8: an 8-bit cache; kPairs: interleaved pairs
template <typename T, int kLanes, bool kFp8, bool kPairs>
__global__ __launch_bounds__(256) void heads_prologue_kernel(const PrologueParams p) {
  typedef typename Vec8<T>::type V8;
  const int lane = threadIdx.x & 63, j = lane & (kLanes - 1);
  const int64_t group = ((int64_t)blockIdx.x * 256 + threadIdx.x) / kLanes;
  const int64_t t = group / p.parts;
  const int part = (int)(group - t * p.parts);
  if (t >= p.num_tokens) return;
  const int64_t pos = p.positions[t];
  if (pos < 0 || pos >= p.table_rows) return;                // a position that the tables do not have: nothing is written
  const int64_t slot = p.slots ? p.slots[t] : -1;
  const bool store = p.cache[0] && slot >= 0 && slot < p.num_pages * p.page_size;
  const SlotAt at = slot_at(store ? slot : 0, store ? p.page_size : 1);
  const bool mine = j * 8 < p.dim;                           // (heads of fewer values than the group has room for)
  const int r = p.rotary, half_lanes = r >> 4;
  const bool turns = j * 8 < r;
  const bool first = j < half_lanes;
  float c[8], s[8];
#pragma unroll
  for (int e = 0; e < 8; e++) { c[e] = 1.f; s[e] = 0.f; }
  if (turns) {
    if constexpr (kPairs) {
      entries4(p.cos + pos * p.cs_st, j * 4, p.table_f32, c);
      entries4(p.sin + pos * p.cs_st, j * 4, p.table_f32, s);
    } else {
      entries(p.cos + pos * p.cs_st, (first ? j : j - half_lanes) * 8, p.table_f32, c);
      entries(p.sin + pos * p.cs_st, (first ? j : j - half_lanes) * 8, p.table_f32, s);
    }
  }
  const int other = (lane & ~(kLanes - 1)) + (first ? j + half_lanes : j - half_lanes);
  const int heads = p.q_heads + (p.cache[0] || p.out[1] ? p.kv_heads : 0) + (p.cache[0] ? p.kv_heads : 0);
  for (int head = part; head < heads; head += p.parts) {
    const int what = head < p.q_heads ? 0 : head < p.q_heads + p.kv_heads ? 1 : 2;
    const int h = head - (what == 0 ? 0 : what == 1 ? p.q_heads : p.q_heads + p.kv_heads);
    if (what > 0 && !store && !(what == 1 && p.out[1])) continue;
    V8 raw;
#pragma unroll
    for (int e = 0; e < 8; e++) raw[e] = (T)0.f;
    if (mine) raw = *(const V8*)(p.src[what] + t * p.src_st[what] + h * p.src_sh[what] + j * 16);
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = (float)raw[e];
    if (what < 2) {
      if (p.gamma[what]) {
        float sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e++) sum += x[e] * x[e];
#pragma unroll
        for (int o = 1; o < kLanes; o <<= 1) sum += __shfl_xor(sum, o, 64);
        const float inv = 1.f / sqrtf(sum / (float)p.dim + p.eps);
        V8 g;
#pragma unroll
        for (int e = 0; e < 8; e++) g[e] = (T)0.f;
        if (mine) g = *(const V8*)(p.gamma[what] + j * 16);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = x[e] * inv * (float)g[e];
      }
      if constexpr (kPairs) {
        if (turns) {
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const float a = x[2 * e], b = x[2 * e + 1];
            x[2 * e] = a * c[e] - b * s[e];
            x[2 * e + 1] = b * c[e] + a * s[e];
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const float y = __shfl(x[e], other, 64);
          if (turns) x[e] = first ? x[e] * c[e] - y * s[e] : x[e] * c[e] + y * s[e];
        }
      }
    }
    V8 y;
#pragma unroll
    for (int e = 0; e < 8; e++) y[e] = (T)x[e];
    if (!mine) continue;
    if (what < 2 && p.out[what]) *(V8*)(p.out[what] + t * p.out_st[what] + h * p.out_sh[what] + j * 16) = y;
    if (what > 0 && store) {
      const int i = what - 1;
      char* dst = p.cache[i] + at.pg * p.c_sp[i] + at.off * p.c_sr[i] + h * p.c_sh[i];
      if constexpr (kFp8) *(u32x2*)(dst + j * 8) = to_e4m3(x, p.scale[i] ? p.scale[i][h] : 1.f);
      else *(V8*)(dst + j * 16) = y;
    }
  }
}

template <typename T, int kLanes>
void launch(const PrologueParams& p, bool fp8, bool pairs, unsigned blocks, hipStream_t st) {
  if (fp8 && pairs) hipLaunchKernelGGL((heads_prologue_kernel<T, kLanes, true, true>), dim3(blocks), dim3(256), 0, st, p);
  else if (fp8) hipLaunchKernelGGL((heads_prologue_kernel<T, kLanes, true, false>), dim3(blocks), dim3(256), 0, st, p);
  else if (pairs) hipLaunchKernelGGL((heads_prologue_kernel<T, kLanes, false, true>), dim3(blocks), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((heads_prologue_kernel<T, kLanes, false, false>), dim3(blocks), dim3(256), 0, st, p);
}

}  // namespace heads
}  // namespace mlahip
using namespace mlahip;

extern "C" int mlahip_qk_norm_rope_cache(
    const void* q, int64_t q_stride_t, int64_t q_stride_h, const void* k, int64_t k_stride_t, int64_t k_stride_h, const void* v,
    int64_t v_stride_t, int64_t v_stride_h, int64_t num_tokens, int32_t q_heads, int32_t kv_heads, int32_t dim, int32_t dtype,
    const void* q_gamma, const void* k_gamma, float eps, const void* cos, const void* sin, int64_t cs_stride, int64_t table_rows,
    int32_t table_dtype, int32_t rotary_dim, int32_t interleaved, const int64_t* positions, const int64_t* slot_mapping,
    void* k_cache, int64_t kc_page_stride, int64_t kc_row_stride, int64_t kc_head_stride, void* v_cache, int64_t vc_page_stride,
    int64_t vc_row_stride, int64_t vc_head_stride, int32_t page_size, int64_t num_pages, int32_t cache_dtype, const float* k_scale,
    const float* v_scale, void* q_out, int64_t qo_stride_t, int64_t qo_stride_h, void* k_out, int64_t ko_stride_t,
    int64_t ko_stride_h, hipStream_t stream) {
  const char* me = "mlahip_qk_norm_rope_cache";
  const bool cached = k_cache || v_cache || slot_mapping, has_k = kv_heads > 0;
  MLA_REQUIRE((q || q_heads == 0) && (q_out || q_heads == 0) && cos && sin && positions && (k || !has_k), MLA_ERR_NULL, "%s: null pointer argument", me);
  MLA_REQUIRE(!cached || (k_cache && v_cache && slot_mapping && v && has_k), MLA_ERR_NULL,
              "%s: a cache write needs keys, values, both caches and a slot mapping", me);
  MLA_REQUIRE(!has_k || cached || k_out, MLA_ERR_NULL, "%s: keys go to a cache or to k_out", me);
  MLA_REQUIRE((dtype == 0 || dtype == 2) && (table_dtype == 0 || table_dtype == 1) && (!cached || cache_dtype == dtype || cache_dtype == 3),
              MLA_ERR_UNSUPPORTED, "%s: inputs bf16 (0) or fp16 (2), tables bf16 or fp32 (1), caches of the inputs' type or e4m3 (3)", me);
  MLA_REQUIRE(num_tokens >= 0 && q_heads >= 0 && kv_heads >= 0 && q_heads + kv_heads >= 1 && dim >= 16 && dim <= 256 && dim % 16 == 0 &&
                  rotary_dim >= 16 && rotary_dim <= dim && rotary_dim % 16 == 0 && table_rows >= 1 && num_tokens < (1ll << 31) &&
                  q_heads <= 65536 && kv_heads <= 65536,
              MLA_ERR_SHAPE, "%s: %lld tokens, %d + %d heads of %d values, %d rotated, tables of %lld positions (heads of 16..256 values and "
              "rotated parts in multiples of 16)", me, (long long)num_tokens, q_heads, kv_heads, dim, rotary_dim, (long long)table_rows);
  MLA_REQUIRE(!cached || (page_size >= 1 && num_pages >= 1), MLA_ERR_SHAPE, "%s: %lld pages of %d", me, (long long)num_pages, page_size);
  const bool fp8 = cached && cache_dtype == 3;
  const int64_t in_strides = q_stride_t | q_stride_h | (has_k ? k_stride_t | k_stride_h : 0) | (cached ? v_stride_t | v_stride_h : 0) |
                             qo_stride_t | qo_stride_h | (k_out ? ko_stride_t | ko_stride_h : 0);
  const int64_t c_strides = cached ? kc_page_stride | kc_row_stride | kc_head_stride | vc_page_stride | vc_row_stride | vc_head_stride : 0;
  const uintptr_t ptrs = (uintptr_t)q | (uintptr_t)k | (cached ? (uintptr_t)v : 0) | (uintptr_t)q_out | (uintptr_t)k_out | (uintptr_t)cos |
                         (uintptr_t)sin | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)q_gamma | (uintptr_t)k_gamma;
  MLA_REQUIRE(in_strides % 8 == 0 && c_strides % 8 == 0 && cs_stride % (table_dtype == 1 ? 4 : 8) == 0 && !(ptrs & 15), MLA_ERR_SHAPE,
              "%s: heads, table and cache rows must be 16-byte aligned (heads of an 8-bit cache: 8)", me);
  if (num_tokens == 0) return MLA_OK;
  heads::PrologueParams p{};
  p.src[0] = (const char*)q; p.src_st[0] = q_stride_t * 2; p.src_sh[0] = q_stride_h * 2;
  p.src[1] = (const char*)k; p.src_st[1] = k_stride_t * 2; p.src_sh[1] = k_stride_h * 2;
  p.src[2] = (const char*)v; p.src_st[2] = v_stride_t * 2; p.src_sh[2] = v_stride_h * 2;
  p.out[0] = (char*)q_out; p.out_st[0] = qo_stride_t * 2; p.out_sh[0] = qo_stride_h * 2;
  p.out[1] = (char*)k_out; p.out_st[1] = ko_stride_t * 2; p.out_sh[1] = ko_stride_h * 2;
  const int es = fp8 ? 1 : 2;
  p.cache[0] = (char*)k_cache; p.c_sp[0] = kc_page_stride * es; p.c_sr[0] = kc_row_stride * es; p.c_sh[0] = kc_head_stride * es;
  p.cache[1] = (char*)v_cache; p.c_sp[1] = vc_page_stride * es; p.c_sr[1] = vc_row_stride * es; p.c_sh[1] = vc_head_stride * es;
  p.gamma[0] = (const char*)q_gamma; p.gamma[1] = (const char*)k_gamma;
  p.scale[0] = k_scale; p.scale[1] = v_scale;
  p.cos = (const char*)cos; p.sin = (const char*)sin; p.cs_st = cs_stride * (table_dtype == 1 ? 4 : 2); p.table_rows = table_rows;
  p.positions = positions; p.slots = slot_mapping;
  p.num_tokens = num_tokens; p.num_pages = num_pages; p.page_size = page_size;
  p.q_heads = q_heads; p.kv_heads = kv_heads; p.dim = dim; p.rotary = rotary_dim; p.table_f32 = table_dtype == 1;
  p.eps = eps;
  const int lanes = dim <= 64 ? 8 : dim <= 128 ? 16 : 32;
  // groups to a token: a wavefront's lanes are full, and few tokens get more groups so that the CUs have work
  const int total = q_heads + (has_k ? kv_heads : 0) + (cached ? kv_heads : 0), per_wave = 64 / lanes;
  int64_t parts = (16384 + num_tokens - 1) / num_tokens;
  parts = parts < per_wave ? per_wave : parts;
  p.parts = (int)(parts < total ? parts : total);
  const int64_t blocks = (num_tokens * p.parts * lanes + 255) / 256;
  MLA_REQUIRE(blocks < (1ll << 31), MLA_ERR_SHAPE, "%s: too many tokens for one launch", me);
#define HEADS_LAUNCH(L)                                                                  \
  if (dtype == 0) heads::launch<__bf16, L>(p, fp8, interleaved != 0, (unsigned)blocks, stream); \
  else heads::launch<_Float16, L>(p, fp8, interleaved != 0, (unsigned)blocks, stream)
  if (lanes == 8) { HEADS_LAUNCH(8); }
  else if (lanes == 16) { HEADS_LAUNCH(16); }
  else { HEADS_LAUNCH(32); }
#undef HEADS_LAUNCH
  return check_launch(me);
}
