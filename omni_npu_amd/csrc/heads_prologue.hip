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
// A group of 8, 16 or 32 lanes holds a head, four pairs a lane (of half pairs its values are four in either half, so that both of a pair
// are the lane's own); the norm's sum goes by lane moves.  A group takes several heads of one token, so that the token's table entries
// and the gains are read once, and asks for the next head's values before it turns this one's; few tokens get more groups, so that the CUs
// have work.
//
// What bounds it is memory, every value read and written once: 16 384 tokens x 64 + 2 x 8 heads of 128 into the 8-bit cache (646 MB) take
// 115 us, 5.6 TB/s (a copy of 2 GiB on this card: 4.94).  2999 tokens x 16 + 2 x 4 heads of 64 (19 MB) take 6.6 us, and 1 token 2.7, 64 tokens 2.8 in
// a graph, which is a launch and two reads one behind the other (slot and position; then table row and values).  Without the next head's values on their
// way 10 786 tokens x 8 + 2 x 8 heads of 256 took 72 us in place of 53; with the first key and value head of a group asked for in front of its queries
// (80 registers in place of 60) 16 384 x 32 + 2 x 8 of 128 took 81 in place of 78.
#include <type_traits>

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

template <typename T> struct Vec4 { typedef T type __attribute__((ext_vector_type(4))); };

// four entries of a table from entry i on
__device__ __forceinline__ f32x4 entries(const char* row, int i, bool f32) {
  if (f32) return *(const f32x4*)(row + i * 4);
  const bf16x4 a = *(const bf16x4*)(row + i * 2);
  return f32x4{(float)a[0], (float)a[1], (float)a[2], (float)a[3]};
}

// Sum over the 8, 16 or 32 lanes of a head: within rows of 16 by data-parallel-primitive moves.
template <int kLanes> __device__ __forceinline__ float lanes_sum(float x) {
  auto add = [&](auto ctrl) { x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xf, 0xf, true)); };
  add(std::integral_constant<int, 0xB1>{});                  // the neighbour, the pair beside, the other half row mirrored,
  add(std::integral_constant<int, 0x4E>{});
  add(std::integral_constant<int, 0x141>{});
  if constexpr (kLanes >= 16) add(std::integral_constant<int, 0x140>{});   // the row mirrored
  if constexpr (kLanes >= 32) x += __shfl_xor(x, 16, 64);
  return x;
}

// x / s to e4m3, saturated: the quotient by the reciprocal and one correction by the remainder (a division is ten instructions a value)
__device__ __forceinline__ uint32_t to_e4m3(const float* x, float s, float inv) {
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; e++) {
    const float v = x[e] * inv, w = __builtin_fmaf(__builtin_fmaf(-v, s, x[e]), inv, v);
    y[e] = __builtin_isinf(v) ? v : w;                       // (no remainder of an infinity)
    y[e] = y[e] != y[e] ? y[e] : fminf(fmaxf(y[e], -448.f), 448.f);
  }
  int w = 0;
  w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], w, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
  return (uint32_t)w;
}

// What is read and written once, past the caches or through them.
template <bool kPast, typename V> __device__ __forceinline__ V take(const void* at) {
  return kPast ? __builtin_nontemporal_load((const V*)at) : *(const V*)at;
}
template <bool kPast, typename V> __device__ __forceinline__ void give(void* at, V x) {
  if constexpr (kPast) __builtin_nontemporal_store(x, (V*)at);
  else *(V*)at = x;
}

// T: the inputs' type; kLanes: lanes of a head; kFp8: an 8-bit cache; kPairs: interleaved pairs; kPast: past the caches
template <typename T, int kLanes, bool kFp8, bool kPairs, bool kPast>
__global__ __launch_bounds__(256) void heads_prologue_kernel(const PrologueParams p) {
  typedef typename Vec4<T>::type V4;
  typedef T V8 __attribute__((ext_vector_type(8)));
  struct Eight { V4 a, b; };                                 // (filled by parts: as 16 bytes the compiler keeps it in LDS, three times the time)
  const int j = threadIdx.x & (kLanes - 1);
  const int64_t group = ((int64_t)blockIdx.x * 256 + threadIdx.x) / kLanes;
  const uint32_t t32 = (uint32_t)group / (uint32_t)p.parts;  // (host: fewer than 2^32 groups)
  const int64_t t = t32;
  const int part = (int)((uint32_t)group - t32 * (uint32_t)p.parts);
  if (t >= p.num_tokens) return;
  const int64_t pos = p.positions[t];
  const int64_t slot = p.slots ? p.slots[t] : -1;
  if (pos < 0 || pos >= p.table_rows) return;                // a position that the tables do not have: nothing is written
  const bool store = p.cache[0] && slot >= 0 && slot < p.num_pages * p.page_size;
  const SlotAt at = slot_at(store ? slot : 0, store ? p.page_size : 1);
  const bool mine = j * 8 < p.dim;                           // (heads of fewer values than the group has room for)
  // A lane's eight values are two fours at a and b.  A lane that turns half pairs has four pairs: 4j .. of the rotated part's first
  // half and 4j .. of its second.  Lanes that do not exist in the head repeat its lane 0.
  const bool turns = j * 8 < p.rotary;
  const int a0 = !mine ? 0 : !kPairs && turns ? j * 4 : j * 8, b0 = !kPairs && turns && mine ? j * 4 + p.rotary / 2 : a0 + 4;
  f32x4 c{}, s{};
  if (turns) {
    c = entries(p.cos + pos * p.cs_st, j * 4, p.table_f32);
    s = entries(p.sin + pos * p.cs_st, j * 4, p.table_f32);
  }
  auto load = [&](const char* at) {
    if constexpr (kPairs) {
      const V8 x = take<kPast, V8>(at + a0 * 2);
      return Eight{__builtin_shufflevector(x, x, 0, 1, 2, 3), __builtin_shufflevector(x, x, 4, 5, 6, 7)};
    } else {
      return Eight{take<kPast, V4>(at + a0 * 2), take<kPast, V4>(at + b0 * 2)};
    }
  };
  auto store8 = [&](char* at, const float* x) {
    V8 y;
#pragma unroll
    for (int e = 0; e < 8; e++) y[e] = (T)x[e];
    if constexpr (kPairs) {
      give<kPast>(at + a0 * 2, y);
    } else {
      give<kPast, V4>(at + a0 * 2, __builtin_shufflevector(y, y, 0, 1, 2, 3));
      give<kPast, V4>(at + b0 * 2, __builtin_shufflevector(y, y, 4, 5, 6, 7));
    }
  };
  auto cache_row = [&](int i, int h) { return p.cache[i] + at.pg * p.c_sp[i] + at.off * p.c_sr[i] + h * p.c_sh[i]; };
  const float inv_dim = 1.f / (float)p.dim;
  auto turned = [&](const Eight& raw, const char* gamma, const Eight& g, float* x) {
#pragma unroll
    for (int e = 0; e < 4; e++) { x[e] = (float)raw.a[e]; x[4 + e] = (float)raw.b[e]; }
    if (gamma) {
      float sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; e++) sum += x[e] * x[e];
      const float inv = __builtin_amdgcn_rsqf(lanes_sum<kLanes>(mine ? sum : 0.f) * inv_dim + p.eps);
#pragma unroll
      for (int e = 0; e < 4; e++) { x[e] *= inv * (float)g.a[e]; x[4 + e] *= inv * (float)g.b[e]; }
    }
    if (!turns) return;                                      // (1 x + 0 y would not be x beside an infinity)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      float &u = kPairs ? x[2 * e] : x[e], &v = kPairs ? x[2 * e + 1] : x[4 + e];
      const float u0 = u, v0 = v;
      u = u0 * c[e] - v0 * s[e];
      v = v0 * c[e] + u0 * s[e];
    }
  };
  // The token's heads in a row: queries, keys, values; this group takes every parts-th of them, the next one's values asked for ahead.
  int head = part;
  {
    const char *gamma = p.gamma[0], *src = p.src[0] + t * p.src_st[0];
    char* out = p.out[0] + t * p.out_st[0];
    Eight g{}, next{};
    if (gamma && head < p.q_heads) g = load(gamma);
    if (head < p.q_heads) next = load(src + head * p.src_sh[0]);
    for (; head < p.q_heads; head += p.parts) {
      const Eight raw = next;
      if (head + p.parts < p.q_heads) next = load(src + (head + p.parts) * p.src_sh[0]);
      float x[8];
      turned(raw, gamma, g, x);
      if (mine) store8(out + head * p.out_sh[0], x);
    }
  }
  const int keys = p.q_heads + (store || p.out[1] ? p.kv_heads : 0);
  if (head < keys) {
    const char *gamma = p.gamma[1], *src = p.src[1] + t * p.src_st[1];
    Eight g{}, next = load(src + (head - p.q_heads) * p.src_sh[1]);
    if (gamma) g = load(gamma);
    for (; head < keys; head += p.parts) {
      const int h = head - p.q_heads;
      const Eight raw = next;
      if (head + p.parts < keys) next = load(src + (h + p.parts) * p.src_sh[1]);
      float x[8];
      turned(raw, gamma, g, x);
      if (!mine) continue;
      if (p.out[1]) store8(p.out[1] + t * p.out_st[1] + h * p.out_sh[1], x);
      if (!store) continue;
      char* dst = cache_row(0, h);
      if constexpr (kFp8) {
        const float sc = p.scale[0] ? p.scale[0][h] : 1.f, inv = 1.f / sc;
        const uint32_t lo = to_e4m3(x, sc, inv), hi = to_e4m3(x + 4, sc, inv);
        if constexpr (kPairs) {
          give<kPast>(dst + a0, u32x2{lo, hi});
        } else {
          give<kPast>(dst + a0, lo);
          give<kPast>(dst + b0, hi);
        }
      } else {
        store8(dst, x);
      }
    }
  }
  if (!store || !mine || head >= keys + p.kv_heads) return;
  // (values are not turned: eight in a row to a lane)
  const char* src = p.src[2] + t * p.src_st[2] + j * 16;
  V8 next = take<kPast, V8>(src + (head - keys) * p.src_sh[2]);
  for (; head < keys + p.kv_heads; head += p.parts) {
    const int h = head - keys;
    const V8 raw = next;
    if (head + p.parts < keys + p.kv_heads) next = take<kPast, V8>(src + (h + p.parts) * p.src_sh[2]);
    char* dst = cache_row(1, h);
    if constexpr (kFp8) {
      float x[8];
#pragma unroll
      for (int e = 0; e < 8; e++) x[e] = (float)raw[e];
      const float sc = p.scale[1] ? p.scale[1][h] : 1.f, inv = 1.f / sc;
      give<kPast>(dst + j * 8, u32x2{to_e4m3(x, sc, inv), to_e4m3(x + 4, sc, inv)});
    } else {
      give<kPast>(dst + j * 16, raw);
    }
  }
}

template <typename T, int kLanes, bool kPast>
void launch(const PrologueParams& p, bool fp8, bool pairs, unsigned blocks, hipStream_t st) {
  if (fp8 && pairs) hipLaunchKernelGGL((heads_prologue_kernel<T, kLanes, true, true, kPast>), dim3(blocks), dim3(256), 0, st, p);
  else if (fp8) hipLaunchKernelGGL((heads_prologue_kernel<T, kLanes, true, false, kPast>), dim3(blocks), dim3(256), 0, st, p);
  else if (pairs) hipLaunchKernelGGL((heads_prologue_kernel<T, kLanes, false, true, kPast>), dim3(blocks), dim3(256), 0, st, p);
  else hipLaunchKernelGGL((heads_prologue_kernel<T, kLanes, false, false, kPast>), dim3(blocks), dim3(256), 0, st, p);
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
  // Groups to a token: a power of two, so that tokens do not straddle workgroups, with four to seven heads each, or three; a group to a head
  // where that leaves CUs without work.  us by heads of a group, 1 / 2 / 3 / 4 / 5 / 6 / 10 / 20: 16 384 tokens x 80 heads of 128 into the 8-bit cache
  // 171 / 132 / 131 / 121 / 120 / 125 / 126 / 136, 48 (16 each) 108 / 92 / 84 / 79 / 79 / 73 / 77 / 78, 10 786 x 24 of 256 77 / 65 / 59 / 56 / 55 / 52 / 54 /
  // 53; 6000 x 48 of 128, 16 bits, 39 / 34 / 32 / 33 / 34 / 33 / 35 / 35; 700 x 48 7.3 / 6.6 / 6.6 / 7.0 / 7.7 / 7.9 / 9.2 / 11.4, 300 x 80 5.2 / 5.3 / 6.1 /
  // 5.8 / 6.0 / 6.9 / 7.5 / 10.7.
  const int total = q_heads + (has_k ? kv_heads : 0) + (cached ? kv_heads : 0);
  p.parts = 1;
  while (p.parts * 8 <= total) p.parts *= 2;
  constexpr int64_t kFew = 8 * 256 * 64;                     // threads of eight wavefronts to a CU
  while (num_tokens * p.parts * lanes < kFew && p.parts * 6 <= total) p.parts *= 2;
  if (num_tokens * p.parts * lanes < kFew) p.parts = total;
  const int64_t blocks = (num_tokens * p.parts * lanes + 255) / 256;
  MLA_REQUIRE(num_tokens * p.parts < (1ll << 32) - 64 && blocks < (1ll << 31), MLA_ERR_SHAPE, "%s: too many tokens for one launch", me);
  // Past the caches from 64 MB of input on, which would not wait in them for the attention behind: us through / past them, 16 384 tokens x 64 + 2 x 8
  // heads of 128 into the 8-bit cache 122 / 114, x 32 + 2 x 8 81 / 74, 6000 x 32 + 2 x 8 (74 MB) 34 / 30, 1674 x 64 + 2 x 8 of 256 (69 MB) 30.5 / 29.3; 16 384 x
  // 8 + 2 x 8 of 64 (50 MB) 23.6 / 24.4, 3000 x 32 + 2 x 8 of 128 (37 MB) 13.7 / 16.3.
  const bool past = num_tokens * total * dim * 2 >= (64ll << 20);
#define HEADS_LAUNCH(L)                                                                                           \
  if (dtype == 0 && past) heads::launch<__bf16, L, true>(p, fp8, interleaved != 0, (unsigned)blocks, stream);    \
  else if (dtype == 0) heads::launch<__bf16, L, false>(p, fp8, interleaved != 0, (unsigned)blocks, stream);      \
  else if (past) heads::launch<_Float16, L, true>(p, fp8, interleaved != 0, (unsigned)blocks, stream);           \
  else heads::launch<_Float16, L, false>(p, fp8, interleaved != 0, (unsigned)blocks, stream)
  if (lanes == 8) { HEADS_LAUNCH(8); }
  else if (lanes == 16) { HEADS_LAUNCH(16); }
  else { HEADS_LAUNCH(32); }
#undef HEADS_LAUNCH
  return check_launch(me);
}
