// Attention of each request's newest tokens over a paged cache of ordinary key and value heads, cut along the cache and joined.
//
//   o[t, h] = sum_j p_j V[j, h / G] / sum_j p_j,   p_j = exp(scale * q[t, h] . K[j, h / G] - m)
// over the keys j that token i of a request's s tokens sees: j <= L - s + i, and j > L - s + i - window where there is a window.
// G = query heads / key heads.  One pass over the keys; m is a running reference of a row, sums are in fp32.
//
// What bounds it is the cache stream: 4 D bytes of a 16-bit cache per key and head against 4 D G multiply-adds, which the matrix
// cores do with most of their rows empty.  So the cache goes from memory straight into LDS (no registers held while it is under
// way), every wavefront has its own ring there (two tiles; the
// waits count copies, so that the next tile's stay under way), and wavefronts do not wait for each other until a piece of a sequence ends.
//
//   work        units of 64 keys of all sequences end to end, cut into equal chunks, one workgroup each (times head and row groups)
//   wavefront   one key head, 16 or 32 query rows (row = token * G + head in the group), tiles of KT keys; with fewer heads than
//               wavefronts several share a head and take every n-th tile
//   S^T = K Q^T v_mfma_f32_16x16x32: 16 keys x 16 rows; a lane has 4 keys of one row
//   O^T += V^T P^T v_mfma_f32_16x16x16: the lane that has a row's 4 probabilities is the one whose operand they are; V transposed by
//               the LDS read.  An 8-bit V comes as pairs of neighbouring dims, even and odd ones into products of their own
//   join        wavefronts of a head through LDS, then chunks of a sequence through the workspace, by a second launch
#include "mla_common.hpp"

namespace mlahip {
namespace gqa {

constexpr int kUnit = 64;                                    // keys of a plan unit
constexpr float kOutgrown = 8.f;                             // log2 units a score may lie above its row's reference

struct Params {
  const char* q; int64_t q_st, q_sh;                         // strides in bytes
  const char *k, *v; int64_t k_sp, k_sr, k_sh, v_sp, v_sr, v_sh;
  const float *k_scale, *v_scale;
  const int32_t* block_table; int64_t bt_stride; int32_t max_blocks;
  const int32_t *seq_lens, *qsl;
  int64_t num_tokens, num_pages;
  int32_t page_shift;                                        // log2 of the page, -1 where it is no power of two
  int32_t page_size, batch, max_q_len, kv_heads, group, window;
  int32_t num_chunks;                                        // 0: a workgroup takes a whole sequence
  int32_t heads_shift;                                       // log2 of the heads of a workgroup
  int32_t head_groups, row_groups;
  float scale_log2;
  char* out; int64_t o_st, o_sh;
  float* lse;                                                // [T, heads] or null
  int32_t* seg_ids;                                          // [batch][2]: first and last partial of a sequence, or -1
  float *part_lse, *part_acc;                                // [slot][kv head][row](, [D])
};

template <typename T> struct Types;
template <> struct Types<__bf16> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  typedef __bf16 v4 __attribute__((ext_vector_type(4)));
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x4 qk(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ f32x4 pv(u32x2 a, u32x2 b, f32x4 c) {
    typedef short s4 __attribute__((ext_vector_type(4)));
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s4, a), __builtin_bit_cast(s4, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ v2 from_e4m3(uint32_t w, bool hi) {
    return hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false);
  }
};
template <> struct Types<_Float16> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  typedef _Float16 v4 __attribute__((ext_vector_type(4)));
  typedef _Float16 v2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x4 qk(v8 a, v8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ f32x4 pv(u32x2 a, u32x2 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(v4, a), __builtin_bit_cast(v4, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ v2 from_e4m3(uint32_t w, bool hi) {
    return hi ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false);
  }
};

// A request's tokens and keys: tokens [q0, q0 + s) of the batch, first key that any token sees, plan units.
struct Seq { int len, q0, s, first, units; };
__device__ __forceinline__ Seq seq_of(const Params& p, int b) {
  Seq x;
  x.len = p.seq_lens[b];
  x.q0 = p.qsl ? p.qsl[b] : b * p.max_q_len;
  x.s = p.qsl ? p.qsl[b + 1] - x.q0 : p.max_q_len;
  x.s = x.s < 0 ? 0 : x.s < p.max_q_len ? x.s : p.max_q_len;
  const int room = p.max_blocks * p.page_size;               // (host: below 2^31)
  x.len = x.len < 0 ? 0 : x.len < room ? x.len : room;
  x.first = 0;
  if (p.window > 0) {
    const int f = x.len - x.s + 1 - p.window;
    x.first = f > 0 ? f : 0;
  }
  const int n = (x.len + kUnit - 1) / kUnit - x.first / kUnit;
  x.units = n > 0 ? n : 1;                                   // (a request without keys: its rows are written all the same)
  return x;
}

// The first unit of chunk c of n over tot units.
__device__ __forceinline__ int chunk_begin(int c, int n, int tot) { return (int)((int64_t)c * tot / n); }

template <typename T, int D, bool kFp8> struct Shape {
  static constexpr int es = kFp8 ? 1 : 2, row_b = D * es;
  static constexpr int kt = 8192 / (2 * row_b) < 16 ? 16 : 8192 / (2 * row_b);   // keys of a tile
  static constexpr int subs = kt / 16, half_b = kt * row_b, copies = half_b / 1024;
  static constexpr int waves = D == 256 ? 4 : 8;
  static constexpr int wave_b = 4 * half_b;                  // two tiles, keys and values
  static constexpr int keys_per_copy = 1024 / row_b, lanes_per_key = row_b / 16;
  // position of granule c (16 bytes) of a key's row: c ^ swz(key): sixteen keys read at one granule hit different banks
  static __device__ __forceinline__ int swz(int key) {
    return row_b >= 256 ? key & 15 : row_b == 128 ? (key >> 1) & 7 : (key >> 2) & 3;
  }
};
// Until at most N of the wavefront's copies are on their way.
template <int N> __device__ __forceinline__ void wait_copies() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
constexpr int kStatFloats = 8 * 2 * 32;                      // maxima and sums of up to 8 wavefronts x 32 rows

template <typename T, int D, bool kFp8, int MT>
__global__ __launch_bounds__((Shape<T, D, kFp8>::waves * 64)) void gqa_split_kernel(const Params p) {
  typedef Shape<T, D, kFp8> Sh;
  typedef Types<T> Ty;
  typedef typename Ty::v8 v8;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  float* stats = (float*)(lds + Sh::waves * Sh::wave_b);     // [2][wave][32]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  const int gr = blockIdx.y, hg = gr % p.head_groups, rg = gr / p.head_groups;
  const int hw = wave & ((1 << p.heads_shift) - 1), kw = wave >> p.heads_shift, kws = Sh::waves >> p.heads_shift;
  const int head = (hg << p.heads_shift) + hw;
  const int row0 = rg * 16 * MT;
  const bool has_head = head < p.kv_heads;
  char* ring = lds + wave * Sh::wave_b;
  const uint32_t ring0 = lds_addr_of(ring);

  // ---- which units are mine ----
  int v_cur = 0, v_end = 0, b = blockIdx.x, v_seq = 0;
  if (p.num_chunks > 0) {
    int tot = 0;
    for (int i = lane; i < p.batch; i += 64) tot += seq_of(p, i).units;
    tot = __builtin_amdgcn_readlane(wave_incl_scan_dpp(tot), 63);
    const int chunks = p.num_chunks < tot ? p.num_chunks : tot;
    if ((int)blockIdx.x >= chunks) return;
    v_cur = __builtin_amdgcn_readfirstlane(chunk_begin(blockIdx.x, chunks, tot));
    v_end = __builtin_amdgcn_readfirstlane(chunk_begin(blockIdx.x + 1, chunks, tot));
    int carry = 0;
    b = 0;
    for (int base = 0; base < p.batch; base += 64) {         // the sequence that holds unit v_cur
      const int i = base + lane;
      const int run = wave_incl_scan_dpp(i < p.batch ? seq_of(p, i).units : 0) + carry;
      const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < p.batch && run <= v_cur));
      if (n > 0) v_seq = __builtin_amdgcn_readlane(run, n - 1);
      b += n;
      carry = __builtin_amdgcn_readlane(run, 63);
    }
  }

  const int rows_max = p.max_q_len * p.group;
  const int64_t k_head = (int64_t)(has_head ? head : 0) * p.k_sh, v_head = (int64_t)(has_head ? head : 0) * p.v_sh;
  const float scale_log2 = p.scale_log2 * (kFp8 && p.k_scale && has_head ? p.k_scale[head] : 1.f);

  for (; p.num_chunks == 0 || v_cur < v_end; b++) {
    if (b >= p.batch) break;
    Seq sq = seq_of(p, b);
    sq.len = __builtin_amdgcn_readfirstlane(sq.len); sq.s = __builtin_amdgcn_readfirstlane(sq.s);
    sq.q0 = __builtin_amdgcn_readfirstlane(sq.q0); sq.first = __builtin_amdgcn_readfirstlane(sq.first);
    sq.units = __builtin_amdgcn_readfirstlane(sq.units);
    int u0 = 0, u1 = sq.units;
    bool whole = true;
    if (p.num_chunks > 0) {
      u0 = v_cur - v_seq;
      u1 = v_end - v_seq < sq.units ? v_end - v_seq : sq.units;
      v_seq += sq.units;
      v_cur = v_seq < v_end ? v_seq : v_end;
      whole = u0 == 0 && u1 == sq.units;
      if (gr == 0 && threadIdx.x == 0) {
        if (u0 == 0) p.seg_ids[2 * b] = whole ? -1 : (int)blockIdx.x + b;
        if (u1 == sq.units && !whole) p.seg_ids[2 * b + 1] = (int)blockIdx.x + b;
      }
    }
    const int rows = sq.s * p.group;
    if (row0 < rows) {
      const int unit0 = sq.first / kUnit;
      int key0 = (unit0 + u0) * kUnit, key1 = (unit0 + u1) * kUnit;
      key0 = key0 > sq.first ? key0 : sq.first / Sh::kt * Sh::kt;
      key1 = key1 < sq.len ? key1 : sq.len;
      const int tiles = key1 > key0 ? (key1 - key0 + Sh::kt - 1) / Sh::kt : 0;
      const int mine = has_head && tiles > kw ? (tiles - kw + kws - 1) / kws : 0;

      // ---- copies of a tile's keys or values into the ring ----
      const int32_t* bt = p.block_table + (int64_t)b * p.bt_stride;
      const int lk = lane / Sh::lanes_per_key, lp = lane % Sh::lanes_per_key;
      // page numbers of the wavefront's next 64 pages, one to a lane
      int have0 = 0, have = 0;
      auto pages_from = [&](int pi) {
        const int at = pi + lane;
        have0 = pi;
        have = bt[at < p.max_blocks ? at : p.max_blocks - 1];
      };
      struct Place { int64_t pg; int off; } place[Sh::subs];
      auto find = [&](int tile) {
#pragma unroll
        for (int s = 0; s < Sh::subs; s++) {
          const int key = key0 + (kw + tile * kws) * Sh::kt + s * 16;
          const int pi = p.page_shift >= 0 ? key >> p.page_shift : (int)((uint32_t)key / (uint32_t)p.page_size);
          place[s].off = __builtin_amdgcn_readfirstlane(p.page_shift >= 0 ? key & (p.page_size - 1) : key - pi * p.page_size);
          if (__builtin_amdgcn_readfirstlane(pi - have0) > 63) pages_from(__builtin_amdgcn_readfirstlane(pi));
          const int64_t pg = __builtin_amdgcn_readlane(have, __builtin_amdgcn_readfirstlane(pi - have0));
          place[s].pg = pg < 0 ? 0 : pg < p.num_pages ? pg : p.num_pages - 1;
        }
      };
      auto copy = [&](int tile, bool values) {
        const char* base = values ? p.v + v_head : p.k + k_head;
        const int64_t sp = values ? p.v_sp : p.k_sp, sr = values ? p.v_sr : p.k_sr;
        const uint32_t to = ring0 + (tile & 1) * 2 * Sh::half_b + (values ? Sh::half_b : 0);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");     // (what was read of the place has arrived)
#pragma unroll
        for (int s = 0; s < Sh::subs; s++) {
          const char* from = base + place[s].pg * sp + (int64_t)place[s].off * sr;
#pragma unroll
          for (int c = 0; c < Sh::copies / Sh::subs; c++) {
            const int kk = c * Sh::keys_per_copy + lk;       // (key of the sixteen)
            const uint32_t at = (uint32_t)kk * (uint32_t)sr + (uint32_t)((lp ^ Sh::swz(kk)) << 4);
            dma16_sv_nt(from, at, to + (s * (Sh::copies / Sh::subs) + c) * 1024);
          }
        }
      };
      if (mine > 0) {
        const int key = key0 + kw * Sh::kt;
        pages_from(__builtin_amdgcn_readfirstlane((int)((uint32_t)key / (uint32_t)p.page_size)));
        find(0);
        copy(0, false);
        copy(0, true);
        if (mine > 1) {
          find(1);
          copy(1, false);
          copy(1, true);
        }
      }

      // ---- the query: row l16 of each row tile, eight dims a step; zeros in rows that do not exist ----
      v8 qf[MT][D / 32];
      int hi[MT], lo[MT], tok[MT];
#pragma unroll
      for (int m = 0; m < MT; m++) {
        const int r = row0 + m * 16 + l16;
        const bool there = r < rows && has_head;
        const int rr = there ? r : 0;
        tok[m] = (int)((uint32_t)rr / (uint32_t)p.group);
        const int64_t t = (int64_t)sq.q0 + tok[m];
        const bool ok = there && t >= 0 && t < p.num_tokens;
        const char* src = p.q + (ok ? t : 0) * p.q_st + (int64_t)((has_head ? head : 0) * p.group + (rr - tok[m] * p.group)) * p.q_sh;
#pragma unroll
        for (int s = 0; s < D / 32; s++) {
          // (an 8-bit key's granule of 16 dims is two steps' operands)
          const int dim = kFp8 ? (s >> 1) * 64 + g * 16 + (s & 1) * 8 : s * 32 + g * 8;
          v8 x;
#pragma unroll
          for (int e = 0; e < 8; e++) x[e] = (T)0.f;
          if (ok) x = *(const v8*)(src + dim * 2);
          qf[m][s] = x;
        }
        hi[m] = sq.len - sq.s + tok[m] + 1;
        lo[m] = p.window > 0 ? hi[m] - p.window : 0;
      }
      // keys that all of the rows see
      const int tok_first = row0 / p.group, tok_last = (row0 + 16 * MT < rows ? row0 + 16 * MT - 1 : rows - 1) / p.group;
      const int all_hi = sq.len - sq.s + tok_first + 1, all_lo = p.window > 0 ? sq.len - sq.s + tok_last + 1 - p.window : 0;

      f32x4 acc[MT][D / 16];
      float m_ref[MT], l_run[MT];
#pragma unroll
      for (int m = 0; m < MT; m++) {
        m_ref[m] = -INFINITY;
        l_run[m] = 0.f;
#pragma unroll
        for (int d = 0; d < D / 16; d++) acc[m][d] = f32x4{0.f, 0.f, 0.f, 0.f};
      }

      for (int i = 0; i < mine; i++) {
        const int tile_key = key0 + (kw + i * kws) * Sh::kt;
        // (younger than the tile's keys: its values, and the next tile's keys and values)
        const bool next = i + 1 < mine, after = i + 2 < mine;
        if (next) wait_copies<3 * Sh::copies>();
        else wait_copies<Sh::copies>();
        const char* kt = ring + (i & 1) * 2 * Sh::half_b;
        const char* vt = kt + Sh::half_b;
        const bool partial = tile_key + Sh::kt > all_hi || tile_key < all_lo;
        // ---- S^T ----
        f32x4 sc[MT][Sh::subs];
#pragma unroll
        for (int s = 0; s < Sh::subs; s++) {
          const char* row = kt + (s * 16 + l16) * Sh::row_b;
          const int sw = Sh::swz(l16);
#pragma unroll
          for (int m = 0; m < MT; m++) sc[m][s] = f32x4{0.f, 0.f, 0.f, 0.f};
          if constexpr (kFp8) {
#pragma unroll
            for (int t = 0; t < D / 64; t++) {
              const u32x4 x = *(const u32x4*)(row + (((t * 4 + g) ^ sw) << 4));
              typename Ty::v2 h[8];
#pragma unroll
              for (int e = 0; e < 4; e++) { h[2 * e] = Ty::from_e4m3(x[e], false); h[2 * e + 1] = Ty::from_e4m3(x[e], true); }
              v8 a, c;
#pragma unroll
              for (int e = 0; e < 4; e++) { a[2 * e] = h[e][0]; a[2 * e + 1] = h[e][1]; c[2 * e] = h[4 + e][0]; c[2 * e + 1] = h[4 + e][1]; }
#pragma unroll
              for (int m = 0; m < MT; m++) {
                sc[m][s] = Ty::qk(a, qf[m][2 * t], sc[m][s]);
                sc[m][s] = Ty::qk(c, qf[m][2 * t + 1], sc[m][s]);
              }
            }
          } else {
#pragma unroll
            for (int t = 0; t < D / 32; t++) {
              const v8 a = *(const v8*)(row + (((t * 4 + g) ^ sw) << 4));
#pragma unroll
              for (int m = 0; m < MT; m++) sc[m][s] = Ty::qk(a, qf[m][t], sc[m][s]);
            }
          }
        }
        if (after) {
          find(i + 2);
          copy(i + 2, false);
        }
        // ---- probabilities against the rows' references ----
        u32x2 pf[MT][Sh::subs];
#pragma unroll
        for (int m = 0; m < MT; m++) {
          float most = -INFINITY;
#pragma unroll
          for (int s = 0; s < Sh::subs; s++) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
              float x = sc[m][s][e] * scale_log2;
              if (partial) {
                const int key = tile_key + s * 16 + 4 * g + e;
                x = key < hi[m] && key >= lo[m] ? x : -INFINITY;
              }
              sc[m][s][e] = x;
              most = fmaxf(most, x);
            }
          }
          if (__builtin_amdgcn_ballot_w64(most > m_ref[m] + kOutgrown)) {
            most = fmaxf(most, __shfl_xor(most, 16, 64));
            most = fmaxf(most, __shfl_xor(most, 32, 64));
            const float next = fmaxf(m_ref[m], most);
            const float f = next > m_ref[m] ? fast_exp2(m_ref[m] - next) : 1.f;
            m_ref[m] = next;
            l_run[m] *= f;
#pragma unroll
            for (int d = 0; d < D / 16; d++) acc[m][d] *= f;
          }
          const float ref = m_ref[m] == -INFINITY ? 0.f : m_ref[m];
#pragma unroll
          for (int s = 0; s < Sh::subs; s++) {
            typename Ty::v4 pr;
#pragma unroll
            for (int e = 0; e < 4; e++) {
              // the probability is rounded to the operand's type, and the rounded one is what the sum counts: the weights that
              // are applied add up to one
              pr[e] = (T)fast_exp2(sc[m][s][e] - ref);
              l_run[m] += (float)pr[e];
            }
            pf[m][s] = __builtin_bit_cast(u32x2, pr);
          }
        }
        if (after) wait_copies<3 * Sh::copies>();
        else if (next) wait_copies<2 * Sh::copies>();
        else wait_copies<0>();
        // ---- O^T += V^T P^T ----
        // A tile with keys that a row does not see is done token by token with those keys' values cleared (0 times what lies there,
        // an infinity or stale NaN, would not be 0), and a lane takes the product of its own row's token.
#pragma unroll
        for (int s = 0; s < Sh::subs; s++) {
          const int vr = s * 16 + 4 * g + (l16 >> 2);
          const char* row = vt + vr * Sh::row_b + (l16 & 1) * 8;
          const int sw = Sh::swz(vr & 15);
          auto values = [&](int d, u32x2* a) {               // operands of dims 16 d .. (8 bits: 32 d .., even and odd)
            const u32x2 x = __builtin_bit_cast(u32x2, lds_read_tr16(row + (((2 * d + ((l16 >> 1) & 1)) ^ sw) << 4)));
            if constexpr (kFp8) {
              // (x: a 16-bit pair of dims of four keys)
              const uint32_t k0 = __builtin_bit_cast(uint32_t, Ty::from_e4m3(x[0], false)), k1 = __builtin_bit_cast(uint32_t, Ty::from_e4m3(x[0], true));
              const uint32_t k2 = __builtin_bit_cast(uint32_t, Ty::from_e4m3(x[1], false)), k3 = __builtin_bit_cast(uint32_t, Ty::from_e4m3(x[1], true));
              a[0] = u32x2{__builtin_amdgcn_perm(k1, k0, 0x05040100), __builtin_amdgcn_perm(k3, k2, 0x05040100)};
              a[1] = u32x2{__builtin_amdgcn_perm(k1, k0, 0x07060302), __builtin_amdgcn_perm(k3, k2, 0x07060302)};
            } else {
              a[0] = x;
            }
          };
          constexpr int kOps = kFp8 ? 2 : 1;
          if (!partial) {
#pragma unroll
            for (int d = 0; d < D / 16 / kOps; d++) {
              u32x2 a[kOps];
              values(d, a);
#pragma unroll
              for (int o = 0; o < kOps; o++)
#pragma unroll
                for (int m = 0; m < MT; m++) acc[m][d * kOps + o] = Ty::pv(a[o], pf[m][s], acc[m][d * kOps + o]);
            }
          } else {
            const int key = tile_key + s * 16 + 4 * g;
            for (int t = tok_first; t <= tok_last; t++) {
              const int t_hi = sq.len - sq.s + t + 1, t_lo = p.window > 0 ? t_hi - p.window : 0;
              u32x2 see;
#pragma unroll
              for (int e = 0; e < 2; e++)
                see[e] = (key + 2 * e < t_hi && key + 2 * e >= t_lo ? 0xffffu : 0u) | (key + 2 * e + 1 < t_hi && key + 2 * e + 1 >= t_lo ? 0xffff0000u : 0u);
#pragma unroll
              for (int d = 0; d < D / 16 / kOps; d++) {
                u32x2 a[kOps];
                values(d, a);
#pragma unroll
                for (int o = 0; o < kOps; o++) {
                  const u32x2 x = {a[o][0] & see[0], a[o][1] & see[1]};
#pragma unroll
                  for (int m = 0; m < MT; m++) {
                    const f32x4 y = Ty::pv(x, pf[m][s], acc[m][d * kOps + o]);
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[m][d * kOps + o][e] = tok[m] == t ? y[e] : acc[m][d * kOps + o][e];
                  }
                }
              }
            }
          }
        }
        if (after) copy(i + 2, true);
      }

      // ---- join of the wavefronts of a head, a row tile at a time, and the rows' results ----
#pragma unroll
      for (int m = 0; m < MT; m++) {
        float l = l_run[m];
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        // granule position in a row: granule ^ row, so that sixteen rows' writes at one granule hit different banks.  Granule:
        // four dims as the accumulator has them (8 bits: every other one of eight)
#pragma unroll
        for (int d = 0; d < D / 16; d++) *(f32x4*)(ring + l16 * (D * 4) + (((d * 4 + g) ^ l16) << 4)) = acc[m][d];
        if (g == 0) {
          stats[wave * 32 + l16] = m_ref[m];
          stats[256 + wave * 32 + l16] = l;
        }
        lds_barrier();
        constexpr int kGran = D / 4;
        const int n_heads = 1 << p.heads_shift, items = n_heads * 16 * kGran;
        for (int it = threadIdx.x; it < items; it += Sh::waves * 64) {
          const int gi = it & (kGran - 1), r16 = (it / kGran) & 15, h = it / (kGran * 16);
          const int r = row0 + m * 16 + r16, hd = (hg << p.heads_shift) + h;
          if (r >= rows || hd >= p.kv_heads) continue;
          float most = -INFINITY;
          for (int k = 0; k < kws; k++) most = fmaxf(most, stats[((k << p.heads_shift) + h) * 32 + r16]);
          const float ref = most == -INFINITY ? 0.f : most;
          float sum = 0.f;
          f32x4 o = {0.f, 0.f, 0.f, 0.f};
          for (int k = 0; k < kws; k++) {
            const int w = (k << p.heads_shift) + h;
            const float mk = stats[w * 32 + r16], lk2 = stats[256 + w * 32 + r16];
            // (a wavefront without keys for the row has zeros and weighs nothing)
            const float wt = mk == -INFINITY ? 0.f : fast_exp2(mk - ref);
            const f32x4 a = *(const f32x4*)(lds + w * Sh::wave_b + r16 * (D * 4) + ((gi ^ r16) << 4));
            sum += wt * lk2;
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] += wt * a[e];
          }
          const float vs = kFp8 && p.v_scale ? p.v_scale[hd] : 1.f;
          const float inv = sum == 0.f ? 0.f : vs / sum;
#pragma unroll
          for (int e = 0; e < 4; e++) o[e] *= inv;
          const float lse = sum == 0.f ? -INFINITY : (most + fast_log2(sum)) * kLn2;
          // dims of the granule: gi = 4 d + g'
          const int dim = kFp8 ? (gi >> 3) * 32 + (gi & 3) * 8 + ((gi >> 2) & 1) : gi * 4, step = kFp8 ? 2 : 1;
          if (whole) {
            const int tk = (int)((uint32_t)r / (uint32_t)p.group);
            const int64_t t = (int64_t)sq.q0 + tk;
            if (t < 0 || t >= p.num_tokens) continue;
            const int qh = hd * p.group + (r - tk * p.group);
            char* dst = p.out + t * p.o_st + (int64_t)qh * p.o_sh;
#pragma unroll
            for (int e = 0; e < 4; e++) *(T*)(dst + (dim + e * step) * 2) = (T)o[e];
            if (p.lse && gi == 0) p.lse[t * (p.kv_heads * p.group) + qh] = lse;
          } else {
            const int64_t slot = ((int64_t)(blockIdx.x + b) * p.kv_heads + hd) * rows_max + r;
#pragma unroll
            for (int e = 0; e < 4; e++) p.part_acc[slot * D + dim + e * step] = o[e];
            if (gi == 0) p.part_lse[slot] = lse;
          }
        }
        lds_barrier();
      }
    }
    if (p.num_chunks == 0) break;
  }
}

// The partials of a sequence's chunks into its rows: a workgroup of four wavefronts for a row; lanes of 4 dims, several partials at once.
template <typename T, int D>
__global__ __launch_bounds__(256) void gqa_join_kernel(const Params p) {
  __shared__ float part[4][D], stat[4][2];
  const int b = blockIdx.y, first = p.seg_ids[2 * b];
  if (first < 0) return;
  const int last = p.seg_ids[2 * b + 1];
  const Seq sq = seq_of(p, b);
  const int rows_max = p.max_q_len * p.group, per_head = rows_max;
  const int hd = blockIdx.x / per_head, r = blockIdx.x % per_head;
  if (r >= sq.s * p.group) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  constexpr int kLanes = D / 4, kPer = 64 / kLanes;          // lanes of a partial; partials of a wavefront at once
  const int sub = lane / kLanes, gi = lane % kLanes;
  const int64_t stride = (int64_t)p.kv_heads * rows_max, base = (int64_t)hd * rows_max + r;
  float most = -INFINITY;
  for (int s = first + lane; s <= last; s += 64) most = fmaxf(most, p.part_lse[s * stride + base]);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
  const float ref = most == -INFINITY ? 0.f : most;
  float sum = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = first + wave * kPer + sub; s <= last; s += 4 * kPer) {
    const float l = p.part_lse[s * stride + base];
    const f32x4 a = *(const f32x4*)(p.part_acc + (s * stride + base) * D + gi * 4);
    const float w = l == -INFINITY ? 0.f : fast_exp2((l - ref) * kLog2e);
    sum += w;
#pragma unroll
    for (int e = 0; e < 4; e++) acc[e] += w * a[e];
  }
#pragma unroll
  for (int o = kLanes; o < 64; o <<= 1) {
    sum += __shfl_xor(sum, o, 64);
#pragma unroll
    for (int e = 0; e < 4; e++) acc[e] += __shfl_xor(acc[e], o, 64);
  }
  if (sub == 0) {
    *(f32x4*)&part[wave][gi * 4] = acc;
    if (gi == 0) stat[wave][0] = sum;
  }
  __syncthreads();
  const int tk = (int)((uint32_t)r / (uint32_t)p.group);
  const int64_t t = (int64_t)sq.q0 + tk;
  if (t < 0 || t >= p.num_tokens) return;
  const int qh = hd * p.group + (r - tk * p.group);
  const float total = stat[0][0] + stat[1][0] + stat[2][0] + stat[3][0];
  for (int d = threadIdx.x; d < D; d += 256) {
    const float o = part[0][d] + part[1][d] + part[2][d] + part[3][d];
    *(T*)(p.out + t * p.o_st + (int64_t)qh * p.o_sh + d * 2) = (T)(total == 0.f ? 0.f : o / total);
  }
  if (p.lse && threadIdx.x == 0) p.lse[t * (p.kv_heads * p.group) + qh] = total == 0.f ? -INFINITY : most + fast_log2(total) * kLn2;
}

template <typename T, int D, bool kFp8, int MT>
int launch(const Params& p, unsigned x, hipStream_t st) {
  typedef Shape<T, D, kFp8> Sh;
  constexpr int bytes = Sh::waves * Sh::wave_b + kStatFloats * 4;
  const int rc = ensure_dynamic_lds((const void*)gqa_split_kernel<T, D, kFp8, MT>, bytes, "mlahip_gqa_decode");
  if (rc != MLA_OK) return rc;
  hipLaunchKernelGGL((gqa_split_kernel<T, D, kFp8, MT>), dim3(x, (unsigned)(p.head_groups * p.row_groups)), dim3(Sh::waves * 64), bytes, st, p);
  if (int e = check_launch("mlahip_gqa_decode")) return e;
  if (p.num_chunks > 0) {
    hipLaunchKernelGGL((gqa_join_kernel<T, D>), dim3((unsigned)(p.kv_heads * p.max_q_len * p.group), (unsigned)p.batch), dim3(256), 0, st, p);
    return check_launch("mlahip_gqa_decode");
  }
  return MLA_OK;
}
template <typename T, int D>
int pick(const Params& p, bool fp8, int mt, unsigned x, hipStream_t st) {
  if (fp8) return mt == 1 ? launch<T, D, true, 1>(p, x, st) : launch<T, D, true, 2>(p, x, st);
  return mt == 1 ? launch<T, D, false, 1>(p, x, st) : launch<T, D, false, 2>(p, x, st);
}
template <typename T>
int pick_dim(const Params& p, int dim, bool fp8, int mt, unsigned x, hipStream_t st) {
  return dim == 64 ? pick<T, 64>(p, fp8, mt, x, st) : dim == 128 ? pick<T, 128>(p, fp8, mt, x, st) : pick<T, 256>(p, fp8, mt, x, st);
}

int64_t slots(int64_t batch, int64_t chunks) { return chunks > 0 ? batch + chunks : 0; }
int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

}  // namespace gqa
}  // namespace mlahip
using namespace mlahip;

extern "C" size_t mlahip_gqa_decode_workspace_bytes(int32_t batch, int32_t max_q_len, int32_t q_heads, int32_t dim, int32_t num_chunks) {
  if (batch <= 0 || max_q_len <= 0 || q_heads <= 0 || dim <= 0 || num_chunks <= 0) return 0;
  const int64_t n = gqa::slots(batch, num_chunks) * max_q_len * q_heads;
  return (size_t)(gqa::align256((int64_t)batch * 8) + gqa::align256(n * 4) + n * dim * 4);
}

extern "C" int mlahip_gqa_decode(const void* q, int64_t q_stride_t, int64_t q_stride_h, int64_t num_tokens, const void* k_cache,
                                 int64_t kc_page_stride, int64_t kc_row_stride, int64_t kc_head_stride, const void* v_cache,
                                 int64_t vc_page_stride, int64_t vc_row_stride, int64_t vc_head_stride, int64_t num_pages,
                                 int32_t page_size, const int32_t* block_table, int64_t bt_stride, int32_t max_blocks,
                                 const int32_t* seq_lens, const int32_t* query_start_loc, int32_t batch, int32_t max_q_len,
                                 int32_t q_heads, int32_t kv_heads, int32_t dim, int32_t dtype, int32_t cache_dtype,
                                 const float* k_scale, const float* v_scale, float scale, int32_t window, void* out,
                                 int64_t out_stride_t, int64_t out_stride_h, float* lse_out, void* workspace, size_t workspace_bytes,
                                 int32_t num_chunks, hipStream_t stream) {
  const char* me = "mlahip_gqa_decode";
  MLA_REQUIRE(q && k_cache && v_cache && block_table && seq_lens && out, MLA_ERR_NULL, "%s: null pointer argument", me);
  MLA_REQUIRE((dtype == 0 || dtype == 2) && (cache_dtype == dtype || cache_dtype == 3), MLA_ERR_UNSUPPORTED,
              "%s: queries bf16 (0) or fp16 (2), caches of their type or e4m3 (3)", me);
  MLA_REQUIRE(dim == 64 || dim == 128 || dim == 256, MLA_ERR_UNSUPPORTED, "%s: heads of %d values (64, 128 or 256)", me, dim);
  MLA_REQUIRE(batch >= 0 && batch <= 65535 && max_q_len >= 1 && kv_heads >= 1 && q_heads >= kv_heads && q_heads % kv_heads == 0 && num_pages >= 1 &&
                  num_tokens >= 0 && num_chunks >= 0 && window >= 0 && max_blocks >= 1 && bt_stride >= max_blocks && (int64_t)max_q_len * q_heads < (1 << 24),
              MLA_ERR_SHAPE, "%s: batch %d, %d tokens each, %d query and %d key heads, %lld pages, %d chunks, window %d", me, batch, max_q_len,
              q_heads, kv_heads, (long long)num_pages, num_chunks, window);
  MLA_REQUIRE(page_size >= 16 && page_size % 16 == 0 && (int64_t)max_blocks * page_size <= 0x7fffff00, MLA_ERR_SHAPE,
              "%s: %d pages of %d tokens a request (pages of a multiple of 16, fewer than 2^31 tokens)", me, max_blocks, page_size);
  const int es = cache_dtype == 3 ? 1 : 2, unit = 16 / es;
  const int64_t c_strides = kc_page_stride | kc_row_stride | kc_head_stride | vc_page_stride | vc_row_stride | vc_head_stride;
  MLA_REQUIRE((q_stride_t | q_stride_h) % 8 == 0 && c_strides % unit == 0 && (out_stride_t | out_stride_h) % 4 == 0 &&
                  !(((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) && !((uintptr_t)out & 7) && kc_row_stride >= 0 &&
                  vc_row_stride >= 0 && kc_row_stride < (1 << 26) && vc_row_stride < (1 << 26),
              MLA_ERR_SHAPE, "%s: heads must be 16-byte aligned (results: 8)", me);
  if (batch == 0 || num_tokens == 0) return MLA_OK;
  const size_t need = mlahip_gqa_decode_workspace_bytes(batch, max_q_len, q_heads, dim, num_chunks);
  MLA_REQUIRE(num_chunks == 0 || (workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= need), MLA_ERR_WORKSPACE,
              "%s: workspace of %zu bytes, %zu are needed", me, workspace ? workspace_bytes : 0, need);
  gqa::Params p{};
  p.q = (const char*)q; p.q_st = q_stride_t * 2; p.q_sh = q_stride_h * 2;
  p.k = (const char*)k_cache; p.k_sp = kc_page_stride * es; p.k_sr = kc_row_stride * es; p.k_sh = kc_head_stride * es;
  p.v = (const char*)v_cache; p.v_sp = vc_page_stride * es; p.v_sr = vc_row_stride * es; p.v_sh = vc_head_stride * es;
  p.k_scale = k_scale; p.v_scale = v_scale;
  p.block_table = block_table; p.bt_stride = bt_stride; p.max_blocks = max_blocks;
  p.seq_lens = seq_lens; p.qsl = query_start_loc;
  p.num_tokens = num_tokens; p.num_pages = num_pages;
  p.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz(page_size) : -1;
  p.page_size = page_size; p.batch = batch; p.max_q_len = max_q_len; p.kv_heads = kv_heads; p.group = q_heads / kv_heads;
  p.window = window; p.num_chunks = num_chunks;
  p.scale_log2 = scale * kLog2e;
  p.out = (char*)out; p.o_st = out_stride_t * 2; p.o_sh = out_stride_h * 2; p.lse = lse_out;
  if (num_chunks > 0) {
    char* ws = (char*)workspace;
    const int64_t n = gqa::slots(batch, num_chunks) * max_q_len * q_heads;
    p.seg_ids = (int32_t*)ws;
    p.part_lse = (float*)(ws + gqa::align256((int64_t)batch * 8));
    p.part_acc = (float*)((char*)p.part_lse + gqa::align256(n * 4));
  }
  const int rows = max_q_len * p.group, mt = rows > 16 ? 2 : 1;
  const int waves = dim == 256 ? 4 : 8;
  // heads of a workgroup: as many as it has wavefronts, where they are a power of two's multiple
  int shift = 0;
  while ((2 << shift) <= waves && kv_heads % (2 << shift) == 0) shift++;
  p.heads_shift = shift;
  p.head_groups = kv_heads >> shift;
  p.row_groups = (rows + 16 * mt - 1) / (16 * mt);
  MLA_REQUIRE((int64_t)p.head_groups * p.row_groups <= 65535, MLA_ERR_SHAPE, "%s: %d head groups x %d row groups", me, p.head_groups, p.row_groups);
  const unsigned x = (unsigned)(num_chunks > 0 ? num_chunks : batch);
  return dtype == 0 ? gqa::pick_dim<__bf16>(p, dim, cache_dtype == 3, mt, x, stream) : gqa::pick_dim<_Float16>(p, dim, cache_dtype == 3, mt, x, stream);
}
