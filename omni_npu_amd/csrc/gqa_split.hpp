// Attention of each request's newest tokens over a paged cache of ordinary key and value heads, cut along the cache and joined.
//
//   o[t, h] = sum_j p_j V[j, h / G] / sum_j p_j,   p_j = exp(scale * q[t, h] . K[j, h / G] - m)
// over the keys j that token i of a request's s tokens sees: j <= L - s + i, and j > L - s + i - window where there is a window.  Tokens drafted as
// a tree (kTree) see the context, j < L - s, and of the s newest keys those whose bits are set in the token's words; with a window the newest of these.
// G = query heads / key heads.  One pass over the keys; m is a running reference of a row, sums are in fp32.
//
// What bounds it is the cache stream where contexts are long (4 D bytes of a 16-bit cache per key and head against 4 D G
// multiply-adds, which the matrix cores do with most of their rows empty), and the length of a wavefront's chain of instructions
// where they are short: it issues one every five clocks.  So a wavefront works alone until a piece of a sequence ends, on tiles of 32
// keys whose loads are all under way while it computes on the tile before.
//
//   work        units of 32 keys of all sequences end to end, cut into equal chunks, one workgroup each (times head and row groups)
//   wavefront   one key head, 16, 32 or 64 query rows (row = token * G + head in the group); several wavefronts share a head and take
//               every n-th tile
//   S^T = K Q^T v_mfma_f32_16x16x32: 16 keys x 16 rows.  The operand is what a lane loads: 16 bytes of the key of its number, so keys go
//               from memory into registers as they are used; a lane gets 4 keys of one row
//   O^T += V^T P^T the same, 32 keys deep: the lane that has a row's 8 probabilities is the one whose operand they are.  Values come into
//               registers in whole rows and go through LDS, whose transposed read makes the operand.  An 8-bit V comes as pairs of
//               neighbouring dims, even and odd ones into products of their own
//   join        wavefronts of a head through LDS, then chunks of a sequence through the workspace, by a second launch
//
// A wait counts loads in their order, so the keys of a tile may be waited for only where it is known what was asked for behind them on every way there:
// each wavefront asks for a first tile, the last tile is a step of its own, and the rare load of page numbers is waited for in its branch.  With
// loads that some ways had and others not, a step waited for its values with its keys: 64 requests x 2000-6000 keys x 8 tokens x 32/8 heads 199 us
// against 193, 4096-8192 keys and trees of 8 tokens 289 against 280; 16 x 3 tokens x 48/3 26.4 against 24.8.
//
// Measured, split and join together: 64 requests x 4096-8192 keys x 32/8 heads of 128 (1630 MB) 251 us, 6.5 TB/s; one of 131 072 x 64/8 90 us,
// 5.9; 128 x 2 tokens x 2048-16 384 keys x 64/8 over the 8-bit cache (2440 MB) 397 us, 6.1; 33 requests x the newest 1024 keys x 16/4 heads of
// 256, pages of 16 (137 MB) 33 us, 4.1: four wavefronts to a CU (a wavefront's sums, keys and values take 300 registers, a second workgroup would
// not fit), five tiles each, and most chunks begin a second sequence.  One request x 1021 keys x 4/1 heads 8.7 us: 6.5 of the split, whose loads
// hang on one another (length, page, keys and values, partial results), 2.2 of the join.
#pragma once
#include <type_traits>

#include "mla_common.hpp"

namespace mlahip {
namespace gqa {

constexpr int kUnit = 32;                                    // keys of a plan unit
constexpr int kTile = 32;                                    // keys of a wavefront's step
// Probabilities go to the products in two operands of the matrix instruction's type: exp2(score - reference) =: x, rounded, and the rest up to
// (1 + 2^-6) x, the probability that both stand for.  More than x, so that the rest is positive whichever way x was rounded: an infinite value gives an
// infinity twice then, and never one less another.  Rounded, the rest is off by (2^-6 + 2^-8) 2^-8 of x in bf16, (2^-6 + 2^-11) 2^-11 in fp16.
constexpr float kWhole = 1.f + 0x1p-6f, kWholeLog2 = 0.02236781302845451f;

struct Params {
  const char *k, *v; int64_t k_sp, v_sp;                     // strides in bytes
  int32_t k_sr, v_sr;
  const int32_t *seq_lens, *qsl, *block_table;
  int64_t bt_stride;
  int32_t max_blocks, num_pages, page_size, page_shift;      // log2 of the page, -1 where it is no power of two
  int32_t batch, max_q_len, kv_heads, group, window;
  int32_t num_chunks;                                        // 0: a workgroup takes a whole sequence
  int32_t spare_units;                                       // by how much a chunk may be longer to be of one sequence
  int32_t heads_shift, head_groups;                          // log2 of the heads of a workgroup
  float scale_log2;
  // (from here on: what a piece's begin and end take)
  int64_t k_sh, v_sh;
  const float *k_scale, *v_scale;
  const char* q; int64_t q_st, q_sh;
  int64_t num_tokens;
  char* out; int64_t o_st, o_sh;
  float* lse;                                                // [T, heads] or null
  int32_t* seg_ids;                                          // [batch][2]: first and last partial of a sequence, or -1
  f32x2* part_lse; float* part_acc;                          // [slot][kv head][row](, [D]); log-sum-exps in log2 units, each as a sum of two
  const uint64_t* visible; int64_t visible_stride; int32_t words;   // trees: [T][words], a token's bits
};

template <typename T> struct Types;
template <> struct Types<__bf16> {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  typedef __bf16 v4 __attribute__((ext_vector_type(4)));
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x4 mm(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t from_e4m3(uint32_t w, bool hi) {
    return __builtin_bit_cast(uint32_t, hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true) : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false));
  }
  static constexpr uint32_t kOnes = 0x3f803f80u;
  // log2 units: how far a row's reference is set below its largest score, and how far above that a later one may lie before it is set anew.
  // Above it here, so that the largest scores' probabilities are 2^-24 to 2^-16: sums over values of any size stay finite.
  static constexpr float kBelow = -24.f, kOutgrown = 8.f;
  static constexpr uint32_t kExp = 0x7f807f80u, kLow = 0x00800080u;   // a number's exponent bits and the lowest of them
};
template <> struct Types<_Float16> {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  typedef _Float16 v4 __attribute__((ext_vector_type(4)));
  typedef _Float16 v2 __attribute__((ext_vector_type(2)));
  static __device__ __forceinline__ f32x4 mm(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t from_e4m3(uint32_t w, bool hi) {
    return __builtin_bit_cast(uint32_t, hi ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false));
  }
  static constexpr uint32_t kOnes = 0x3c003c00u;
  // Probabilities of 2^13 to 2^15 for the largest scores: an fp16 below 2^-14 loses bits, and one below 2^-25 is none.  8192 keys that are worth
  // 2^-26 each beside one key are 2^-13 of the result; with 1 for the largest they were left out of it.  (Setting references anew more often:
  // 64 x 4096-8192 keys x 32/8 heads 263.5 us / 263.6, 33 x 1024 x 16/4 of 256 35.7 / 35.9.)
  static constexpr float kBelow = 13.f, kOutgrown = 2.f;
  static constexpr uint32_t kExp = 0x7c007c00u, kLow = 0x04000400u;
};

// A request's tokens and keys: the first s of its tokens, [q0, q0 + s) of the batch, are done (s <= max_q_len, however many it has); token i sees
// keys below key_0 + i (a tree's tokens: the context ends at key_0, the request's first token's key, however far below 0); plan units.
struct Seq { int len, q0, s, key_0, units; };
__device__ __forceinline__ int first_key(const Params& p, int key_0) {
  return p.window > 0 && key_0 > p.window ? key_0 - p.window : 0;
}
template <bool kTree>
__device__ __forceinline__ Seq seq_from(const Params& p, int len, int q0, int q1) {
  Seq x;
  x.q0 = q0;
  const int room = p.max_blocks * p.page_size;               // (host: at most 2^30)
  x.len = len < 0 ? 0 : len < room ? len : room;
  // (where a request has more tokens than keys, those of its first ones that are done see none either way)
  const int done = kTree && p.words * 64 > p.max_q_len ? p.words * 64 : p.max_q_len;
  const int most = x.len + done, tokens = q1 <= q0 ? 0 : (uint32_t)q1 - (uint32_t)q0 < (uint32_t)most ? q1 - q0 : most;
  x.s = tokens < p.max_q_len ? tokens : p.max_q_len;
  x.key_0 = x.len - tokens + (kTree ? 0 : 1);
  const int n = (x.len + kUnit - 1) / kUnit - first_key(p, x.key_0) / kUnit;
  x.units = n > 0 ? n : 1;                                   // (a request without keys: its rows are written all the same)
  return x;
}
// (lanes of sequences of their own, or a uniform b: scalar loads)
template <bool kTree>
__device__ __forceinline__ Seq seq_of(const Params& p, int b) {
  if (p.qsl) return seq_from<kTree>(p, p.seq_lens[b], p.qsl[b], p.qsl[b + 1]);
  return seq_from<kTree>(p, p.seq_lens[b], b * p.max_q_len, (b + 1) * p.max_q_len);
}
typedef const __attribute__((address_space(4))) int32_t* ConstPtr;
template <bool kTree>
__device__ __forceinline__ Seq seq_at(const Params& p, int b) {
  if (p.qsl) return seq_from<kTree>(p, ((ConstPtr)p.seq_lens)[b], ((ConstPtr)p.qsl)[b], ((ConstPtr)p.qsl)[b + 1]);
  return seq_from<kTree>(p, ((ConstPtr)p.seq_lens)[b], b * p.max_q_len, (b + 1) * p.max_q_len);
}

// Units of a chunk: tot over n, upwards.  (Below 2^21 the quotient's distance from the next integer is at least 0.5 / n, and the
// product's error is below that.)
__device__ __forceinline__ int chunk_units(int tot, int n) {
  tot += n - 1;
  return tot < (1 << 21) ? (int)(((float)tot + 0.5f) * __builtin_amdgcn_rcpf((float)n)) : (int)((uint32_t)tot / (uint32_t)n);
}

// A piece's log-sum-exp, its reference and the sum's logarithm, as what the sum of both is rounded to and what that leaves: at 2^20 one float alone would be off
// by 4 % of the piece's weight, and beyond 2^25 pieces of one key and of thousands would weigh the same.
__device__ __forceinline__ f32x2 lse_of(float ref, float log_sum) {
  const float hi = ref + log_sum, b = hi - ref, lo = (ref - (hi - b)) + (log_sum - b);
  return f32x2{hi, fabsf(hi) < INFINITY ? lo : 0.f};
}

// A page as a buffer, and 16 bytes out of it that are read once: at the lane's offset and a scalar one.  (Host: no page takes 2^31 bytes.)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t page_at(const char* base, int page, int64_t stride, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)(base + (int64_t)page * stride), 0, bytes, 0x00027000);
}
__device__ __forceinline__ u32x4 load_nt(__amdgpu_buffer_rsrc_t from, int lane_offset, int offset) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(from, lane_offset, offset, 2));
}

// Four wavefronts to a workgroup instead of eight: where a wavefront's sums, queries and the tile under way do not fit half of a SIMD's
// registers (32 rows of 128 with 16-bit keys in eight spill: 128 requests x 2000 keys x 64/8 heads, 4 tokens each, 244 us against 135).
constexpr bool few_waves(int rows, int dim, int element_bytes) { return dim == 256 || rows == 64 || (rows == 32 && dim == 128 && element_bytes == 2); }

template <typename T, int D, bool kFp8, int MT> struct Shape {
  static constexpr int es = kFp8 ? 1 : 2, row_b = D * es;
  static constexpr int gran = row_b / 64;                    // loads of sixteen keys: a lane's granules (16 bytes) of its key
  static constexpr int v_loads = kTile * row_b / 1024, keys_per_load = 1024 / row_b, lanes_per_key = row_b / 16;
  static constexpr int waves = few_waves(16 * MT, D, es) ? 4 : 8;
  static constexpr int ops = kFp8 ? 2 : 1;                   // operands of one transposed read
  static constexpr int join_b = 16 * D * 4, tile_b = kTile * row_b;
  static constexpr int wave_b = join_b > tile_b ? join_b : tile_b;
  static constexpr int stat_floats = waves * 2 * 16 * MT + 8 + waves * 16 * MT * 2;   // references, sums, flags, results' addresses
  static constexpr int lds_b = waves * wave_b + stat_floats * 4;                         // (a tree's words behind them)
  // position of granule c of a key's row in LDS: c ^ swz(key), so that rows written and read together hit different banks
  static __device__ __forceinline__ int swz(int key) {
    return row_b >= 256 ? key & 15 : row_b == 128 ? (key >> 1) & 7 : (key >> 2) & 3;
  }
};

// (a pointer out of arguments loaded so is said to be in global memory: flat accesses wait for the LDS as well)
#define GLOBAL __attribute__((address_space(1)))
// The arguments again, to be loaded here: what a piece's begin and end take would hold scalar registers throughout its loop.
typedef const __attribute__((address_space(4))) Params* ParamsPtr;
__device__ __forceinline__ ParamsPtr reload() {
  ParamsPtr p = (ParamsPtr)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return p;
}

// What a tree's tokens see of tiles that hold keys of the request's own tokens, kept in LDS as a word of 32 keys for each tile and token.
constexpr int kMostWords = 8, kTreeTiles = 2 * kMostWords + 1;
__device__ __forceinline__ uint32_t bits_to(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }
// How many of a token's first n bits are set (n: at most 64 * words); word: its words, by their number.
template <typename F> __device__ __forceinline__ int bits_below(F word, int n) {
  int sum = 0;
  for (int w = 0; w * 64 < n; w++) {
    const uint64_t x = word(w);
    sum += __builtin_popcountll(n - w * 64 < 64 ? x & ((1ull << (n - w * 64)) - 1) : x);
  }
  return sum;
}
__device__ __forceinline__ int bits_below(const GLOBAL uint64_t* row, int n) {
  return bits_below([&](int w) { return row[w]; }, n);
}
// The 32 keys from key0 on (key0 + 32 > ctx): the context's, below ctx, and those of the token's bits that are keys of the request's, below len; of
// the bits the lowest ``drop`` ones are in front of the window.
template <typename F> __device__ __forceinline__ uint32_t tree_word(F word, int words, int key0, int ctx, int len, int drop) {
  const int j = key0 > ctx ? key0 - ctx : 0, w = j >> 6, r = j & 63;
  uint32_t x = 0;
  if (w < words) {
    uint64_t y = word(w) >> r;
    if (r > 32 && w + 1 < words) y |= word(w + 1) << (64 - r);
    x = (uint32_t)y;
    if (drop > 0)
      for (int n = drop - bits_below(word, j); n > 0 && x; n--) x &= x - 1;
  }
  if (ctx > key0) x = x << (ctx - key0) | bits_to(ctx - key0);
  return x & bits_to(len - key0);
}

template <bool kTree, typename T, int D, bool kFp8, int MT>
__global__ __launch_bounds__((Shape<T, D, kFp8, MT>::waves * 64)) void gqa_split_kernel(const Params p) {
  typedef Shape<T, D, kFp8, MT> Sh;
  typedef Types<T> Ty;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  float* stats = (float*)(lds + Sh::waves * Sh::wave_b);     // [wave][row] references, then sums; [wave] a piece has to be done again
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int l16 = lane & 15, g = lane >> 4;
  int hg = blockIdx.y, rg = 0;
  if (p.head_groups != (int)gridDim.y) { rg = hg / p.head_groups; hg -= rg * p.head_groups; }
  const int hw = wave & ((1 << p.heads_shift) - 1), kw = wave >> p.heads_shift, kws_shift = (Sh::waves == 8 ? 3 : 2) - p.heads_shift, kws = 1 << kws_shift;
  const int head = (hg << p.heads_shift) + hw;
  const int row0 = rg * 16 * MT;
  char* mine_lds = lds + wave * Sh::wave_b;

  // page numbers of the wavefront's next 64 pages, one to a lane; where the request is known, its first ones, before its length is
  int have0 = 0, have = 0;
  auto pages_from = [&](int b, int pi) {
    const int at = pi + lane;
    have0 = pi;
    have = p.block_table[(int64_t)b * p.bt_stride + (at < p.max_blocks ? at : p.max_blocks - 1)];
  };

  // ---- which units are mine ----
  int v_cur = 0, v_end = 0, b = blockIdx.x, v_seq = 0;
  Seq lane_seq{};
  const bool in_lanes = p.num_chunks > 0 && p.batch <= 64 && p.batch > 1;    // a lane keeps a sequence
  if (p.num_chunks > 0 && p.batch == 1) {                    // (nothing to look for)
    pages_from(0, 0);
    const int tot = seq_at<kTree>(p, 0).units, size = __builtin_amdgcn_readfirstlane(chunk_units(tot, p.num_chunks));
    v_cur = blockIdx.x * size;
    v_end = v_cur + size < tot ? v_cur + size : tot;
    if (v_cur >= tot) return;
    b = 0;
  } else if (p.num_chunks > 0) {
    int ends = 0, tot = 0;
    if (in_lanes) {
      if (lane < p.batch) lane_seq = seq_of<kTree>(p, lane);
      ends = wave_incl_scan_dpp(lane_seq.units);
      tot = __builtin_amdgcn_readlane(ends, 63);
    } else {
      for (int i = lane; i < p.batch; i += 64) tot += seq_of<kTree>(p, i).units;
      tot = __builtin_amdgcn_readlane(wave_incl_scan_dpp(tot), 63);
    }
    int size = __builtin_amdgcn_readfirstlane(chunk_units(tot, p.num_chunks));
    // Chunks of one sequence each, where they are few units longer for it: the start of a second piece costs more.
    const int whole_size = in_lanes && p.num_chunks > p.batch ? __builtin_amdgcn_readfirstlane(chunk_units(tot, p.num_chunks - p.batch)) : 0x7fffffff;
    if (whole_size <= size + p.spare_units) {
      const int mine = chunk_units(lane_seq.units, whole_size);
      const int chunk_ends = wave_incl_scan_dpp(mine);        // (lanes without a sequence: no units)
      b = __builtin_popcountll(__builtin_amdgcn_ballot_w64(lane < p.batch && chunk_ends <= (int)blockIdx.x));
      if (b >= p.batch) return;
      if (b > 0) v_seq = __builtin_amdgcn_readlane(ends, b - 1);
      v_cur = v_seq + ((int)blockIdx.x - (b > 0 ? __builtin_amdgcn_readlane(chunk_ends, b - 1) : 0)) * whole_size;
      const int seq_end = __builtin_amdgcn_readlane(ends, b);
      v_end = v_cur + whole_size < seq_end ? v_cur + whole_size : seq_end;
    } else {
    v_cur = blockIdx.x * size;
    v_end = v_cur + size < tot ? v_cur + size : tot;
    if (v_cur >= tot) return;
    if (in_lanes) {                                          // the sequence that holds unit v_cur
      b = __builtin_popcountll(__builtin_amdgcn_ballot_w64(lane < p.batch && ends <= v_cur));
      if (b > 0) v_seq = __builtin_amdgcn_readlane(ends, b - 1);
    } else {
      int carry = 0;
      b = 0;
      for (int base = 0; base < p.batch; base += 64) {
        const int i = base + lane;
        const int run = wave_incl_scan_dpp(i < p.batch ? seq_of<kTree>(p, i).units : 0) + carry;
        const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < p.batch && run <= v_cur));
        if (n > 0) v_seq = __builtin_amdgcn_readlane(run, n - 1);
        b += n;
        carry = __builtin_amdgcn_readlane(run, 63);
      }
    }
    }
  }

  if (p.num_chunks == 0) pages_from(b, 0);
  do {
    if (b >= p.batch) break;
    Seq sq;
    if (in_lanes) {
      sq.len = __builtin_amdgcn_readlane(lane_seq.len, b); sq.q0 = __builtin_amdgcn_readlane(lane_seq.q0, b);
      sq.s = __builtin_amdgcn_readlane(lane_seq.s, b); sq.key_0 = __builtin_amdgcn_readlane(lane_seq.key_0, b);
      sq.units = __builtin_amdgcn_readlane(lane_seq.units, b);
    } else {
      sq = seq_at<kTree>(p, b);
    }
    int u0 = 0, u1 = sq.units;
    bool whole = true;
    if (p.num_chunks > 0) {
      u0 = v_cur - v_seq;
      u1 = v_end - v_seq < sq.units ? v_end - v_seq : sq.units;
      v_seq += sq.units;
      v_cur = v_seq < v_end ? v_seq : v_end;
      whole = u0 == 0 && u1 == sq.units;
      if (blockIdx.y == 0 && threadIdx.x == 0) {
        GLOBAL int32_t* ids = (GLOBAL int32_t*)reload()->seg_ids + 2 * b;
        if (u0 == 0) ids[0] = whole ? -1 : (int)blockIdx.x + b;
        if (u1 == sq.units && !whole) ids[1] = (int)blockIdx.x + b;
      }
    }
    const int rows = sq.s * p.group;
    if (row0 < rows) {
      const int first_seen = first_key(p, sq.key_0), unit0 = first_seen / kUnit;
      int key0 = (unit0 + u0) * kUnit, key1 = (unit0 + u1) * kUnit;
      key0 = key0 > first_seen ? key0 : first_seen & ~(kTile - 1);
      key1 = key1 < sq.len ? key1 : sq.len;
      const int tiles = key1 > key0 ? (key1 - key0 + kTile - 1) / kTile : 0;
      const int mine = tiles > kw ? (tiles - kw + kws - 1) >> kws_shift : 0;

      // ---- where keys lie ----
      auto page_of = [&](int key) { return __builtin_amdgcn_readfirstlane(p.page_shift >= 0 ? key >> p.page_shift : (int)((uint32_t)key / (uint32_t)p.page_size)); };
      struct Place { int page, row; };
      auto place_of = [&](int key) {                         // (sixteen keys from a multiple of sixteen on: one page)
        const int pi = page_of(key);
        if ((uint32_t)(pi - have0) > 63u) {                  // (in front of them where a piece is begun again)
          pages_from(b, pi);
          asm volatile("" : "+v"(have));                     // (waited for here: behind the branch it would be with every tile, and so all loads)
        }
        const int pg = __builtin_amdgcn_readlane(have, pi - have0);
        return Place{pg < 0 ? 0 : pg < p.num_pages ? pg : p.num_pages - 1, key - pi * p.page_size};
      };
      const ParamsPtr first = reload();
      const char *k_head = p.k + (int64_t)head * first->k_sh, *v_head = p.v + (int64_t)head * first->v_sh;
      // A load's address: the page's (a buffer's base), the row's (a scalar) and the lane's own offset, none of them a lane's work per load
      const int lk = lane / Sh::lanes_per_key, lp = lane % Sh::lanes_per_key;
      const int k_off = l16 * p.k_sr + g * 16, v_off = lk * p.v_sr + lp * 16;
      u32x4 kr[2][Sh::gran], vr[Sh::v_loads];
      Place at[2];
      // (Loads that some wavefronts make and some do not would be waited for with all that follow them: one without tiles makes them too, of the first
      // tile's place, in a buffer of no bytes.)
      const int kw_from = mine > 0 ? kw : 0, readable = mine > 0 ? 0x7fffffff : 0;
      auto ask_keys = [&](int i) {
        const int key = key0 + (kw_from + i * kws) * kTile;
#pragma unroll
        for (int s = 0; s < 2; s++) {
          // (a page of a multiple of 32 holds both sixteens)
          at[s] = s == 1 && (p.page_size & 16) == 0 ? Place{at[0].page, at[0].row + 16} : place_of(key + s * 16);
          const __amdgpu_buffer_rsrc_t from = page_at(k_head, at[s].page, p.k_sp, readable);
#pragma unroll
          for (int c = 0; c < Sh::gran; c++) kr[s][c] = load_nt(from, k_off + c * 64, at[s].row * p.k_sr);
        }
      };
      auto ask_values = [&]() {
#pragma unroll
        for (int s = 0; s < 2; s++) {
          const __amdgpu_buffer_rsrc_t from = page_at(v_head, at[s].page, p.v_sp, readable);
#pragma unroll
          for (int n = 0; n < Sh::v_loads / 2; n++)
            vr[s * (Sh::v_loads / 2) + n] = load_nt(from, v_off, (at[s].row + n * Sh::keys_per_load) * p.v_sr);
        }
      };

      // the rows' tokens
      int tok_first = 0, tok_last = 0;
      if (p.max_q_len > 1) {
        tok_first = (int)((uint32_t)row0 / (uint32_t)p.group);
        tok_last = (int)((uint32_t)((row0 + 16 * MT < rows ? row0 + 16 * MT : rows) - 1) / (uint32_t)p.group);
      }
      uint32_t* tree_words = (uint32_t*)(stats + Sh::stat_floats);   // [token][tile]
      const int tree_tile0 = sq.key_0 & ~(kTile - 1);        // first key of the first tile that is not the context's alone
      const int tree_row = 2 * p.words + 2;                  // its tiles, and how many keys of a window are left to the context
      auto visible_of = [&](int token) {
        const ParamsPtr at = reload();
        const int64_t t = (int64_t)sq.q0 + token;
        return (const GLOBAL uint64_t*)at->visible + (t >= 0 && t < at->num_tokens ? t : 0) * at->visible_stride;
      };
      // how many keys of a window are left to the context, below 0: how many bits are in front of the window
      const int own = sq.len - sq.key_0;
      auto window_left = [&](const GLOBAL uint64_t* row) { return p.window - bits_below(row, own < 64 * p.words ? own : 64 * p.words); };
      auto tile_bits = [&](int token, int tile_key) {        // without the window's begin
        const int n = (tile_key - tree_tile0) / kTile;       // (both multiples)
        return tile_key < tree_tile0 ? 0xffffffffu : n < tree_row - 1 ? tree_words[(token - tok_first) * tree_row + n] : 0u;
      };

      // ---- the query: row l16 of each row tile, eight dims a step; zeros in rows that do not exist ----
      u32x4 qf[MT][D / 32];
      int hi[MT], lo[MT], tok[MT];
      auto load_queries = [&] {
#pragma unroll
        for (int m = 0; m < MT; m++) {
          const int r = row0 + m * 16 + l16;
          const bool there = r < rows;
          const int rr = there ? r : kTree ? row0 : 0;
          tok[m] = p.max_q_len == 1 ? 0 : (int)((uint32_t)rr / (uint32_t)p.group);
          const int64_t t = (int64_t)sq.q0 + tok[m];
          const bool ok = there && t >= 0 && t < first->num_tokens;
          const GLOBAL char* src = (const GLOBAL char*)first->q + (ok ? t : 0) * first->q_st + (int64_t)(head * p.group + (rr - tok[m] * p.group)) * first->q_sh;
#pragma unroll
          for (int s = 0; s < D / 32; s++) {
            // (an 8-bit key's granule of 16 dims is two steps' operands)
            const int dim = kFp8 ? (s >> 1) * 64 + g * 16 + (s & 1) * 8 : s * 32 + g * 8;
            qf[m][s] = ok ? *(const GLOBAL u32x4*)(src + dim * 2) : u32x4{0u, 0u, 0u, 0u};
          }
        }
      };
      // A tree's bits are asked for with the table and the queries, in front of the first keys and values, and looked at while these are under way: a
      // load that is waited for behind them waits for them as well.  One word: a thread's of all tiles that it is in.
      uint64_t word = 0;
      const int word_of = (int)threadIdx.x >> 2;
      if (kTree && p.words == 1) word = *visible_of(tok_first + word_of <= tok_last ? tok_first + word_of : tok_last);
      load_queries();
      if (p.num_chunks == 0 ? p.window > 0 : p.batch > 1) pages_from(b, page_of(key0 + kw_from * kTile));
      if constexpr (!kTree) {
#pragma unroll
        for (int m = 0; m < MT; m++) {
          hi[m] = sq.key_0 + tok[m];
          lo[m] = p.window > 0 ? hi[m] - p.window : 0;
        }
      }
      int only = -1;                                         // the token that a pass is for, where the piece is done token by token
      while (true) {
      if constexpr (kTree) asm volatile("" : "+v"(word), "+v"(have));   // (waited for here)
      __builtin_amdgcn_sched_barrier(0);
      ask_keys(0);
      ask_values();
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (kTree) {
        const int items = (tok_last - tok_first + 1) * tree_row;
        if (only < 0 && p.words == 1) {
          const int n = (int)threadIdx.x & 3, over = p.window > 0 ? bits_below([&](int) { return word; }, own < 64 ? own : 64) - p.window : 0;
          const uint32_t bits = tree_word([&](int) { return word; }, 1, tree_tile0 + n * kTile, sq.key_0, sq.len, over);
          if ((int)threadIdx.x < items) tree_words[threadIdx.x] = n == 3 ? (uint32_t)-over : bits;
        } else if (only < 0) {
          for (int it = threadIdx.x; it < items; it += Sh::waves * 64) {
            const int k = it / tree_row, n = it - k * tree_row;
            const GLOBAL uint64_t* row = visible_of(tok_first + k);
            const int left = p.window > 0 ? window_left(row) : 0;
            const uint32_t bits = tree_word([&](int w) { return row[w]; }, p.words, tree_tile0 + n * kTile, sq.key_0, sq.len, -left);
            tree_words[it] = n == tree_row - 1 ? (uint32_t)left : bits;
          }
        }
        lds_barrier();
#pragma unroll
        for (int m = 0; m < MT; m++) {
          const int left = p.window > 0 ? (int)tree_words[(tok[m] - tok_first + 1) * tree_row - 1] : 0;
          lo[m] = p.window > 0 ? sq.key_0 - (left > 0 ? left : 0) : 0;
        }
      }
      const int t0 = only < 0 ? tok_first : only, t1 = only < 0 ? tok_last : only;
      // (a tree's: the context that every token sees, and the keys that there are)
      const int all_hi = sq.key_0 + (kTree ? 0 : t0), any_hi = kTree ? sq.len : sq.key_0 + t1;
      const int all_lo = p.window > 0 ? (kTree ? any_hi : sq.key_0 + t1) - p.window : 0;
      int any_lo = p.window > 0 ? all_hi - p.window : 0;
      if constexpr (kTree) {
        if (p.window > 0 && t0 == t1) {                      // (one token's: where its own window begins)
          const int left = (int)tree_words[(t0 - tok_first + 1) * tree_row - 1];
          any_lo = sq.key_0 - (left > 0 ? left : 0);
        }
      }
      uint32_t odd = 0;
      const float scale_log2 = first->scale_log2 * (kFp8 && first->k_scale ? ((const GLOBAL float*)first->k_scale)[head] : 1.f);

      f32x4 acc[MT][D / 16], sum[MT];                        // sum: of the probabilities, by a product with ones
      float m_ref[MT];
#pragma unroll
      for (int m = 0; m < MT; m++) {
        m_ref[m] = -INFINITY;
        sum[m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int d = 0; d < D / 16; d++) acc[m][d] = f32x4{0.f, 0.f, 0.f, 0.f};
      }
      // (the last tile by itself: where the next one's loads may be missing the compiler waits for them with those that it means)
      auto step = [&](int i, auto kMore) __attribute__((always_inline)) {
        const int tile_key = key0 + (kw + i * kws) * kTile;
        const bool partial = tile_key + kTile > all_hi || tile_key < all_lo;
        // ---- S^T ----
        f32x4 sc[MT][2];
#pragma unroll
        for (int s = 0; s < 2; s++) {
#pragma unroll
          for (int m = 0; m < MT; m++) sc[m][s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < Sh::gran; c++) {
            const u32x4 x = kr[s][c];
            if constexpr (kFp8) {
              u32x4 a, z;
#pragma unroll
              for (int e = 0; e < 2; e++) {
                a[2 * e] = Ty::from_e4m3(x[e], false); a[2 * e + 1] = Ty::from_e4m3(x[e], true);
                z[2 * e] = Ty::from_e4m3(x[2 + e], false); z[2 * e + 1] = Ty::from_e4m3(x[2 + e], true);
              }
#pragma unroll
              for (int m = 0; m < MT; m++) sc[m][s] = Ty::mm(z, qf[m][2 * c + 1], Ty::mm(a, qf[m][2 * c], sc[m][s]));
            } else {
#pragma unroll
              for (int m = 0; m < MT; m++) sc[m][s] = Ty::mm(x, qf[m][c], sc[m][s]);
            }
          }
        }
        // (the barriers for the scheduler keep the next tile's loads behind the last use of the registers they go to)
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (kMore()) ask_keys(i + 1);
        __builtin_amdgcn_sched_barrier(0);
        // ---- probabilities against the rows' references ----
        u32x4 pf[MT], pl[MT];
#pragma unroll
        for (int m = 0; m < MT; m++) {
          float most = -INFINITY;
#pragma unroll
          for (int s = 0; s < 2; s++)
#pragma unroll
            for (int e = 0; e < 4; e++) sc[m][s][e] *= scale_log2;
          if (kTree && partial) {
            const uint32_t bits = (tile_bits(tok[m], tile_key) & ~bits_to(lo[m] - tile_key)) >> 4 * g;
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
              for (int e = 0; e < 4; e++) sc[m][s][e] = bits & 1u << (s * 16 + e) ? sc[m][s][e] : -INFINITY;
          } else if (partial) {
#pragma unroll
            for (int s = 0; s < 2; s++)
#pragma unroll
              for (int e = 0; e < 4; e++) {
                const int key = tile_key + s * 16 + 4 * g + e;
                sc[m][s][e] = key < hi[m] && key >= lo[m] ? sc[m][s][e] : -INFINITY;
              }
          }
#pragma unroll
          for (int s = 0; s < 2; s++)
#pragma unroll
            for (int e = 0; e < 4; e++) most = fmaxf(most, sc[m][s][e]);
          // (a difference: beyond 2^24 a sum would round to a larger one, and fp16 ends at 2^16)
          if (__builtin_amdgcn_ballot_w64(most - m_ref[m] > Ty::kBelow + Ty::kOutgrown)) {
            most = fmaxf(most, __shfl_xor(most, 16, 64));
            most = fmaxf(most, __shfl_xor(most, 32, 64));
            const float next = fmaxf(m_ref[m], most - (fabsf(most) < 0x1p20f ? Ty::kBelow : 0.f));
            const float f = next > m_ref[m] ? fast_exp2(m_ref[m] - next) : 1.f;
            m_ref[m] = next;
            sum[m] *= f;
#pragma unroll
            for (int d = 0; d < D / 16; d++) acc[m][d] *= f;
          }
          const float ref = m_ref[m] == -INFINITY ? 0.f : m_ref[m];
#pragma unroll
          for (int s = 0; s < 2; s++) {
            // One operand alone would be off by 2^-8 of a probability in bf16, 2^-11 in fp16: as much as a result's own rounding.  The second
            // takes up to 1.5 % of the time with 16 and 32 rows (64 x 4096-8192 keys x 32/8 heads 252 us / 254), with 64 rows, which the products
            // bound, 2-9 (64 x 4 tokens x 2000-6000 keys x 64/4 of 128 125 / 127.5, e4m3 95.5 / 103), long prompts 20.  The sum counts what the
            // products take: the weights that are applied add up to one.
            typename Ty::v4 pr, rest;
#pragma unroll
            for (int e = 0; e < 4; e++) {
              // (not one operation with the product above: scores of 2^25 and more lie further from their unrounded ones than fp16 reaches)
#pragma clang fp contract(off)
              const float x = fast_exp2(sc[m][s][e] - ref);
              pr[e] = (T)x;
              rest[e] = (T)__builtin_fmaf(x, kWhole, -(float)pr[e]);
            }
            const u32x2 w = __builtin_bit_cast(u32x2, pr), z = __builtin_bit_cast(u32x2, rest);
            pf[m][2 * s] = w[0];
            pf[m][2 * s + 1] = w[1];
            pl[m][2 * s] = z[0];
            pl[m][2 * s + 1] = z[1];
          }
          const u32x4 ones = {Ty::kOnes, Ty::kOnes, Ty::kOnes, Ty::kOnes};
          sum[m] = Ty::mm(ones, pl[m], Ty::mm(ones, pf[m], sum[m]));
        }
        // the values have arrived: into LDS (a wavefront's LDS operations keep their order: the reads of the tile before are done)
        __builtin_amdgcn_sched_barrier(0);
        // Keys that no row sees are cleared (0 times what lies there, an infinity or stale NaN, would not be 0).  A value that is not
        // finite and is seen by some rows only is noted: the piece is done again then, token by token.
        if (partial) {
          uint32_t seen = 0xffffffffu;                       // (a tree's token, where the rows are one token's: what it sees)
          if constexpr (kTree) {
            if (t0 == t1) seen = tile_bits(t0, tile_key) >> lk;
          }
#pragma unroll
          for (int n = 0; n < Sh::v_loads; n++) {
            const int key = tile_key + n * Sh::keys_per_load + lk;
            const bool in = key >= any_lo && key < any_hi && (!kTree || (seen & 1u << n * Sh::keys_per_load));
#pragma unroll
            for (int e = 0; e < 4; e++) vr[n][e] = in ? vr[n][e] : 0u;
          }
          if (t0 != t1) {
#pragma unroll
            for (int n = 0; n < Sh::v_loads; n++)
#pragma unroll
              for (int e = 0; e < 4; e++)
                // (all exponent bits set, 8 bits: all bits but the sign, carry into the bit above them)
                odd |= kFp8 ? ((vr[n][e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u : ((vr[n][e] & Ty::kExp) + Ty::kLow) & 0x80008000u;
          }
        }
#pragma unroll
        for (int n = 0; n < Sh::v_loads; n++) {
          const int row = n * Sh::keys_per_load + lk;
          *(u32x4*)(mine_lds + row * Sh::row_b + ((lp ^ Sh::swz(row & 15)) << 4)) = vr[n];
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (kMore()) ask_values();
        __builtin_amdgcn_sched_barrier(0);
        // ---- O^T += V^T P^T ----
        const int v_row = 4 * g + (l16 >> 2), sw = Sh::swz(v_row);
        const char* v_at = mine_lds + v_row * Sh::row_b + (l16 & 1) * 8;
        auto values = [&](int d, u32x4* a) {                 // operands of dims 16 d .. (8 bits: 32 d .., even and odd)
          const char* from = v_at + (((2 * d + ((l16 >> 1) & 1)) ^ sw) << 4);
          const u32x2 x0 = __builtin_bit_cast(u32x2, lds_read_tr16(from)), x1 = __builtin_bit_cast(u32x2, lds_read_tr16(from + 16 * Sh::row_b));
          if constexpr (kFp8) {
            uint32_t w[8];                                   // (a pair of dims of a key each)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              w[2 * e] = Ty::from_e4m3(x0[e], false); w[2 * e + 1] = Ty::from_e4m3(x0[e], true);
              w[4 + 2 * e] = Ty::from_e4m3(x1[e], false); w[4 + 2 * e + 1] = Ty::from_e4m3(x1[e], true);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
              a[0][e] = __builtin_amdgcn_perm(w[2 * e + 1], w[2 * e], 0x05040100);
              a[1][e] = __builtin_amdgcn_perm(w[2 * e + 1], w[2 * e], 0x07060302);
            }
          } else {
            a[0] = u32x4{x0[0], x0[1], x1[0], x1[1]};
          }
        };
#pragma unroll
        for (int d = 0; d < D / 16 / Sh::ops; d++) {
          u32x4 a[Sh::ops];
          values(d, a);
#pragma unroll
          for (int o = 0; o < Sh::ops; o++)
#pragma unroll
            for (int m = 0; m < MT; m++) acc[m][d * Sh::ops + o] = Ty::mm(a[o], pf[m], acc[m][d * Sh::ops + o]);
#pragma unroll
          for (int o = 0; o < Sh::ops; o++)
#pragma unroll
            for (int m = 0; m < MT; m++) acc[m][d * Sh::ops + o] = Ty::mm(a[o], pl[m], acc[m][d * Sh::ops + o]);
        }
      };
      for (int i = 0; i + 1 < mine; i++) step(i, std::true_type{});
      if (mine > 0) step(mine - 1, std::false_type{});

      // ---- join of the wavefronts of a head ----
      const bool several = only < 0 && tok_first != tok_last, again = several && __builtin_amdgcn_ballot_w64(odd != 0) != 0;
      bool by_token = false;
      const ParamsPtr last = reload();
      int tid = threadIdx.x;                                 // (hidden: the addresses below are not worked out, and kept, in front of the loop)
      asm volatile("" : "+v"(tid));
      const int jl = tid & 63, j16 = jl & 15, jg = jl >> 4;
      constexpr int kRows = 16 * MT, kGran = D / 4, kThreads = Sh::waves * 64;
      float *refs = stats, *sums = refs + Sh::waves * kRows, *flags = sums + Sh::waves * kRows;
      int64_t* places = (int64_t*)(flags + 8);               // [row][head]
      const int rows_here = rows - row0 < kRows ? rows - row0 : kRows;
      if (jl < 16) {
#pragma unroll
        for (int m = 0; m < MT; m++) {
          refs[wave * kRows + m * 16 + jl] = m_ref[m];
          sums[wave * kRows + m * 16 + jl] = sum[m][0];
        }
        if (jl == 0) flags[wave] = again ? 1.f : 0.f;
      }
      // Sixteen rows' sums go through LDS at a time.  Granule position in a row: granule ^ row, so that sixteen rows' writes at one granule
      // hit different banks.  Granule: four dims as the accumulator has them (8 bits: every other one of eight)
      auto put = [&](const f32x4 (&a)[D / 16]) {
        char* to = mine_lds + j16 * (D * 4);
#pragma unroll
        for (int d = 0; d < D / 16; d++) *(f32x4*)(to + (((d * 4 + jg) ^ j16) << 4)) = a[d];
      };
      if constexpr (MT == 1) put(acc[0]);
      lds_barrier();
      if (several) {
        for (int k = 0; k < Sh::waves; k++) by_token |= flags[k] != 0.f;
      }
      // What is a row's, by kWs wavefronts of a head: their weights, and where the result goes (0: nowhere).
      auto row_of = [&](auto kWs, int h, int rr, bool first_dims, float* wt) {
        constexpr int kw_n = decltype(kWs)::value;
        const int r = row0 + rr, hd = (hg << p.heads_shift) + h;
        float part[kw_n], most = -INFINITY, total = 0.f;
#pragma unroll
        for (int k = 0; k < kw_n; k++) {
          const int w = (k << p.heads_shift) + h;
          wt[k] = refs[w * kRows + rr];
          part[k] = sums[w * kRows + rr];
        }
#pragma unroll
        for (int k = 0; k < kw_n; k++) most = fmaxf(most, wt[k]);
        const float base = most == -INFINITY ? 0.f : most;
#pragma unroll
        for (int k = 0; k < kw_n; k++) {
          wt[k] = fast_exp2(wt[k] - base);                   // (a wavefront without keys for the row has zeros and weighs nothing)
          total += wt[k] * part[k];
        }
        const float vs = kFp8 && last->v_scale ? ((const GLOBAL float*)last->v_scale)[hd] : 1.f;
        const float inv = total == 0.f ? 0.f : vs / total;
#pragma unroll
        for (int k = 0; k < kw_n; k++) wt[k] *= inv;
        const int tk = p.max_q_len == 1 ? 0 : (int)((uint32_t)r / (uint32_t)p.group), qh = hd * p.group + (r - tk * p.group);
        const int64_t t = (int64_t)sq.q0 + tk;
        if ((only >= 0 && tk != only) || (whole && (t < 0 || t >= last->num_tokens))) return (char*)nullptr;
        const f32x2 lse2 = total == 0.f ? f32x2{-INFINITY, 0.f} : lse_of(most, fast_log2(total) - kWholeLog2);
        if (whole) {
          if (last->lse && first_dims) ((GLOBAL float*)last->lse)[t * (p.kv_heads * p.group) + qh] = lse2[0] * kLn2;
          return last->out + t * last->o_st + (int64_t)qh * last->o_sh;
        }
        const int64_t slot = ((int64_t)(blockIdx.x + b) * p.kv_heads + hd) * (p.max_q_len * p.group) + r;
        if (first_dims) ((GLOBAL f32x2*)last->part_lse)[slot] = lse2;
        return (char*)(last->part_acc + slot * D);
      };
      // Four dims of a row.  Granule gi = 4 d + g'
      const int gi = tid & (kGran - 1), dim = kFp8 ? (gi >> 3) * 32 + (gi & 3) * 8 + ((gi >> 2) & 1) : gi * 4;
      auto from = [&](int k, int h, int r16) {
        return *(const f32x4*)(lds + ((k << p.heads_shift) + h) * Sh::wave_b + r16 * (D * 4) + ((gi ^ r16) << 4));
      };
      auto add = [&](auto kWs, const f32x4* a, const float* wt, char* place) {
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < decltype(kWs)::value; k++)
#pragma unroll
          for (int e = 0; e < 4; e++) o[e] += wt[k] * a[k][e];
        if (!place) return;
        if (whole) {
          GLOBAL T* dst = (GLOBAL T*)place + dim;
          if constexpr (kFp8) {
#pragma unroll
            for (int e = 0; e < 4; e++) dst[2 * e] = (T)o[e];
          } else {
            typename Ty::v4 y;
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = (T)o[e];
            *(GLOBAL typename Ty::v4*)dst = y;
          }
        } else {
          GLOBAL float* dst = (GLOBAL float*)place + dim;
          if constexpr (kFp8) {
#pragma unroll
            for (int e = 0; e < 4; e++) dst[2 * e] = o[e];
          } else {
            *(GLOBAL f32x4*)dst = o;
          }
        }
      };
      auto by_waves = [&](auto f) {
        if (kws == 1) f(std::integral_constant<int, 1>{});
        else if (kws == 2) f(std::integral_constant<int, 2>{});
        else if (Sh::waves == 4 || kws == 4) f(std::integral_constant<int, 4>{});
        else f(std::integral_constant<int, 8>{});
      };
      const int of_row = tid / kGran, heads_of = 1 << p.heads_shift;
      if (by_token) {
        lds_barrier();                                       // (the flags have been read)
      } else if (MT == 1 && rows_here * heads_of <= kThreads / kGran) {
        // Few enough for a granule to a thread: each works its row's weights out by itself.  (1 x 64 keys x 4/1 heads of 128 5.1 us, by a row to
        // a thread first 5.8; the other way round, 1 x 26 keys x 64/4 heads of 256, four heads to a workgroup, 13.6 and 10.6.)
        by_waves([&](auto n) {
          const int h = of_row & (heads_of - 1), r16 = of_row >> p.heads_shift;
          float wt[decltype(n)::value];
          f32x4 a[decltype(n)::value];
          if (r16 >= rows_here) return;
#pragma unroll
          for (int k = 0; k < decltype(n)::value; k++) a[k] = from(k, h, r16);
          add(n, a, wt, row_of(n, h, r16, gi == 0, wt));
        });
        lds_barrier();
      } else {
        // first what is a row's, a row to a thread (a thousand clocks of one instruction after the other), then the sums
        by_waves([&](auto n) {
          for (int it = tid; it < rows_here * heads_of; it += kThreads) {
            const int h = it & (heads_of - 1), rr = it >> p.heads_shift;
            float wt[decltype(n)::value];
            places[it] = (int64_t)row_of(n, h, rr, true, wt);
#pragma unroll
            for (int k = 0; k < decltype(n)::value; k++) refs[((k << p.heads_shift) + h) * kRows + rr] = wt[k];
          }
        });
#pragma unroll 1
        for (int m = 0; m < MT; m++) {
          if (m * 16 >= rows_here) break;
          if constexpr (MT > 1) {
#pragma unroll
            for (int k = 0; k < MT; k++)
              if (k == m) put(acc[k]);
          }
          lds_barrier();
          const int there = rows_here - m * 16 < 16 ? rows_here - m * 16 : 16;
          by_waves([&](auto n) {
#pragma unroll 2
            for (int it = of_row; it < there * heads_of; it += kThreads / kGran) {
              const int h = it & (heads_of - 1), r16 = it >> p.heads_shift;
              float wt[decltype(n)::value];
              f32x4 a[decltype(n)::value];
#pragma unroll
              for (int k = 0; k < decltype(n)::value; k++) {
                wt[k] = refs[((k << p.heads_shift) + h) * kRows + m * 16 + r16];
                a[k] = from(k, h, r16);
              }
              add(n, a, wt, (char*)places[m * 16 * heads_of + it]);
            }
          });
          lds_barrier();
        }
      }
      if (by_token) only = tok_first;
      else if (only < 0 || ++only > tok_last) break;
      }
    }
    b++;
  } while (v_cur < v_end);
}

// The partials of a sequence's chunks into its rows, by the weights exp2(lse_k - max lse): lanes of 4 dims, kWaves wavefronts for a row, each with
// several partials at once; or (0) the lanes of several rows in a wavefront, each of which goes through its partials, four at once.  Both go by their
// own partials' largest log-sum-exp, so that all that is read of them is asked for together.  Rows side by side are few workgroups, and a request that has most
// of a batch's keys has most of its partials: those of kMany and more get a wavefront for each row behind the others, by what each request has.
// They are kept in log2 units: behind a product the compiler would subtract from the unrounded one, which is far off beyond 2^32.
// Bound by the launch and two dependent reads: 2.2 us for 4 rows of 32 partials by four wavefronts; 64 requests x 256 rows of 128 dims of 2 partials 5.8,
// 8 x 3840 of 3 10 (47 MB), where a wavefront for a row took 8.8 and 13; still ahead of it with 8 partials to a request, 194.8 / 195.2 with the
// attention.  With the attention, all rows side by side / a wavefront to each of those of many: one request of 131 072 keys and 63 of 100, 32/8 heads of 64,
// 86.7 / 65.1, of 128, 124.1 / 116.6; batches of equal lengths pay up to 1 us for looking.  A weight is at most 2^-24 (kFar), so that sums over results of
// any size stay finite.
constexpr float kFar = 24.f;
constexpr int kMany = 16;
template <bool kTree, typename T, int D, int kWaves>
__device__ __forceinline__ void join_rows(const Params& p, int b, int first, int last, int item, int w) {
  __shared__ float part[4][D], stat[4][3];
  constexpr int kLanes = D / 4, kPer = 64 / kLanes;          // lanes of a partial; partials, or rows, of a wavefront at once
  constexpr int kApart = kWaves == 0 ? 1 : kWaves * kPer;    // between a lane's partials
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane / kLanes, gi = lane % kLanes;
  const int rows_max = p.max_q_len * p.group;
  const Seq sq = seq_at<kTree>(p, b);
  if (first < 0) return;
  const int hd = (int)((uint32_t)item / (uint32_t)rows_max), r = item - hd * rows_max;
  const bool there = hd < p.kv_heads && r < sq.s * p.group;
  const int64_t stride = (int64_t)p.kv_heads * rows_max, base = there ? (int64_t)hd * rows_max + r : 0;
  f32x2 most = {-INFINITY, 0.f};
  float sum = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  // A difference of two; the larger of each part, which neither lies above; what to weigh by.  (The differences first: beyond 2^23 a sum with kFar rounds.)
  auto above = [](f32x2 x, f32x2 y) { return (x[0] - y[0]) + (x[1] - y[1]); };
  auto higher = [](f32x2 x, f32x2 y) { return f32x2{fmaxf(x[0], y[0]), fmaxf(x[1], y[1])}; };
  auto base_of = [](f32x2 x) { return f32x2{x[0] == -INFINITY ? 0.f : x[0], x[1]}; };
  for (int s0 = first + w; s0 <= last; s0 += 4 * kApart) {
    f32x2 l[4], next = most;
    f32x4 a[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const int s = s0 + k * kApart, at = s <= last ? s : last;
      l[k] = p.part_lse[at * stride + base];
      a[k] = *(const f32x4*)(p.part_acc + (at * stride + base) * D + gi * 4);
      l[k] = s <= last ? l[k] : f32x2{-INFINITY, 0.f};
    }
#pragma unroll
    for (int k = 0; k < 4; k++) next = higher(next, l[k]);
    const f32x2 ref = base_of(next);
    const float f = fast_exp2(above(most, ref));             // (nothing so far: zeros)
    sum *= f;
#pragma unroll
    for (int e = 0; e < 4; e++) acc[e] *= f;
    most = next;
#pragma unroll
    for (int k = 0; k < 4; k++) {
      const float wt = fast_exp2(above(l[k], ref) - kFar);
      sum += wt;
#pragma unroll
      for (int e = 0; e < 4; e++) acc[e] += wt == 0.f ? 0.f : wt * a[k][e];
    }
  }
  // the wavefront's partials side by side, then the row's wavefronts
  f32x2 top = most;
  if constexpr (kWaves > 0) {
#pragma unroll
    for (int o = kLanes; o < 64; o <<= 1) top = higher(top, f32x2{__shfl_xor(top[0], o, 64), __shfl_xor(top[1], o, 64)});
    const float f = fast_exp2(above(most, base_of(top)));
    sum *= f;
#pragma unroll
    for (int e = 0; e < 4; e++) acc[e] *= f;
#pragma unroll
    for (int o = kLanes; o < 64; o <<= 1) {
      sum += __shfl_xor(sum, o, 64);
#pragma unroll
      for (int e = 0; e < 4; e++) acc[e] += __shfl_xor(acc[e], o, 64);
    }
  }
  if constexpr (kWaves > 1) {
    if (sub == 0) {
      *(f32x4*)&part[wave][gi * 4] = acc;
      if (gi == 0) { stat[wave][0] = top[0]; stat[wave][1] = top[1]; stat[wave][2] = sum; }
    }
    __syncthreads();
    if (wave != 0) return;
    f32x2 all = {-INFINITY, 0.f};
#pragma unroll
    for (int k = 0; k < kWaves; k++) all = higher(all, f32x2{stat[k][0], stat[k][1]});
    const f32x2 ref = base_of(all);
    sum = 0.f;
    acc = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kWaves; k++) {
      const float wt = fast_exp2(above(f32x2{stat[k][0], stat[k][1]}, ref));
      const f32x4 a = *(const f32x4*)&part[k][gi * 4];
      sum += wt * stat[k][2];
#pragma unroll
      for (int e = 0; e < 4; e++) acc[e] += wt * a[e];
    }
    top = all;
  }
  if (!there || (kWaves > 0 && sub != 0)) return;
  const int tk = p.max_q_len == 1 ? 0 : (int)((uint32_t)r / (uint32_t)p.group);
  const int64_t t = (int64_t)sq.q0 + tk;
  if (t < 0 || t >= p.num_tokens) return;
  const int qh = hd * p.group + (r - tk * p.group);
  typename Types<T>::v4 y;
#pragma unroll
  for (int e = 0; e < 4; e++) y[e] = (T)(sum == 0.f ? 0.f : acc[e] / sum);
  *(typename Types<T>::v4*)(p.out + t * p.o_st + (int64_t)qh * p.o_sh + gi * 8) = y;
  if (p.lse && gi == 0) p.lse[t * (p.kv_heads * p.group) + qh] = sum == 0.f ? -INFINITY : (top[0] + (top[1] + fast_log2(sum) + kFar)) * kLn2;
}

template <bool kTree, typename T, int D, int kWaves>
__global__ __launch_bounds__(256) void gqa_join_kernel(const Params p, int many) {
  constexpr int kPer = 256 / D;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), sub = lane / (D / 4);
  const ConstPtr ids = (ConstPtr)p.seg_ids;
  if constexpr (kWaves > 0) {
    const int b = blockIdx.y;
    join_rows<kTree, T, D, kWaves>(p, b, ids[2 * b], ids[2 * b + 1], blockIdx.x * (4 / kWaves) + wave / kWaves, wave % kWaves * kPer + sub);
  } else if ((int)blockIdx.y < p.batch) {
    const int b = blockIdx.y, first = ids[2 * b], last = ids[2 * b + 1];
    if (first < 0 || last - first < many) join_rows<kTree, T, D, 0>(p, b, first, last, (blockIdx.x * 4 + wave) * kPer + sub, 0);
  } else {
    // a wavefront for a row of the which-th request of many partials, if there is one
    const int at = ((int)blockIdx.y - p.batch) * (int)gridDim.x + (int)blockIdx.x, groups = (p.kv_heads * p.max_q_len * p.group + 3) / 4;
    int which = at / groups;
    const int item = (at - which * groups) * 4 + wave;
    typedef int32_t i32x2 __attribute__((ext_vector_type(2)));
    for (int base = 0; base < p.batch; base += 64) {
      const i32x2 x = ((const GLOBAL i32x2*)p.seg_ids)[base + lane < p.batch ? base + lane : p.batch - 1];
      uint64_t found = __builtin_amdgcn_ballot_w64(base + lane < p.batch && x[0] >= 0 && x[1] - x[0] >= many);
      const int n = __builtin_popcountll(found);
      if (which >= n) {
        which -= n;
        continue;
      }
      for (; which > 0; which--) found &= found - 1;
      const int l = __builtin_ctzll(found);
      join_rows<kTree, T, D, 1>(p, base + l, __builtin_amdgcn_readlane(x[0], l), __builtin_amdgcn_readlane(x[1], l), item, sub);
      return;
    }
  }
}

template <bool kTree, typename T, int D>
int launch_join(const char* me, const Params& p, hipStream_t st) {
  // the rows of a wavefront side by side where the chunks leave a few partials to a request, four wavefronts to a row where they leave many
  const int items = p.kv_heads * p.max_q_len * p.group;
  if (p.num_chunks > 8 * p.batch) {
    hipLaunchKernelGGL((gqa_join_kernel<kTree, T, D, 4>), dim3((unsigned)items, (unsigned)p.batch), dim3(256), 0, st, p, 0);
  } else {
    // (each of a request's partials but its first begins a chunk: there are so many of kMany)
    const int64_t x = (items + 1024 / D - 1) / (1024 / D), more = ((p.num_chunks - 1) / kMany * (int64_t)((items + 3) / 4) + x - 1) / x;
    const bool fits = D < 256 && p.batch + more <= 65535;    // (heads of 256: a wavefront has one row either way)
    hipLaunchKernelGGL((gqa_join_kernel<kTree, T, D, 0>), dim3((unsigned)x, (unsigned)(p.batch + (fits ? more : 0))), dim3(256), 0, st, p,
                       fits ? kMany : 0x7fffffff);
  }
  return check_launch(me);
}
template <bool kTree, typename T, int D, bool kFp8, int MT>
int launch(const char* me, const Params& p, int row_groups, unsigned x, hipStream_t st) {
  typedef Shape<T, D, kFp8, MT> Sh;
  constexpr int bytes = Sh::lds_b + (kTree ? 16 * MT * (kTreeTiles + 1) * 4 : 0);
  const int rc = ensure_dynamic_lds((const void*)gqa_split_kernel<kTree, T, D, kFp8, MT>, bytes, me);
  if (rc != MLA_OK) return rc;
  hipLaunchKernelGGL((gqa_split_kernel<kTree, T, D, kFp8, MT>), dim3(x, (unsigned)(p.head_groups * row_groups)), dim3(Sh::waves * 64), bytes, st, p);
  if (int e = check_launch(me)) return e;
  return p.num_chunks > 0 ? launch_join<kTree, T, D>(me, p, st) : MLA_OK;
}
// 64 rows to a wavefront are for heads of up to 128: wider ones' sums of as many rows do not fit its registers.
template <bool kTree, typename T, int D, bool kFp8>
int pick(const char* me, const Params& p, int mt, int row_groups, unsigned x, hipStream_t st) {
  if constexpr (D < 256) {
    if (mt == 4) return launch<kTree, T, D, kFp8, 4>(me, p, row_groups, x, st);
  }
  return mt == 1 ? launch<kTree, T, D, kFp8, 1>(me, p, row_groups, x, st) : launch<kTree, T, D, kFp8, 2>(me, p, row_groups, x, st);
}
template <bool kTree, typename T, int D>
int pick(const char* me, const Params& p, bool fp8, int mt, int row_groups, unsigned x, hipStream_t st) {
  return fp8 ? pick<kTree, T, D, true>(me, p, mt, row_groups, x, st) : pick<kTree, T, D, false>(me, p, mt, row_groups, x, st);
}
template <bool kTree, typename T>
int pick(const char* me, const Params& p, int dim, bool fp8, int mt, int row_groups, unsigned x, hipStream_t st) {
  return dim == 64 ? pick<kTree, T, 64>(me, p, fp8, mt, row_groups, x, st) : dim == 128 ? pick<kTree, T, 128>(me, p, fp8, mt, row_groups, x, st)
                                                                                       : pick<kTree, T, 256>(me, p, fp8, mt, row_groups, x, st);
}

// Partial results that there may be: of one piece none, no request is cut.
inline int64_t slots(int64_t batch, int64_t chunks) { return chunks > 1 ? batch + chunks : 0; }
inline int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }
inline size_t workspace_need(int32_t batch, int32_t max_q_len, int32_t q_heads, int32_t dim, int32_t num_chunks) {
  if (batch <= 0 || max_q_len <= 0 || q_heads <= 0 || dim <= 0 || num_chunks <= 0) return 0;
  const int64_t n = slots(batch, num_chunks) * max_q_len * q_heads;
  return (size_t)(align256((int64_t)batch * 8) + align256(n * 8) + n * dim * 4);
}

// gqa_wide.hip: 128 rows to a workgroup.
int launch_wide_rows(const char* me, const Params& p, int dtype, int dim, bool fp8, unsigned x, hipStream_t st);

// The checks and the launches of both entry points.
template <bool kTree>
int run(const char* me, const void* q, int64_t q_stride_t, int64_t q_stride_h, int64_t num_tokens, const void* k_cache,
                                 int64_t kc_page_stride, int64_t kc_row_stride, int64_t kc_head_stride, const void* v_cache,
                                 int64_t vc_page_stride, int64_t vc_row_stride, int64_t vc_head_stride, int64_t num_pages,
                                 int32_t page_size, const int32_t* block_table, int64_t bt_stride, int32_t max_blocks,
                                 const int32_t* seq_lens, const int32_t* query_start_loc, int32_t batch, int32_t max_q_len,
                                 int32_t q_heads, int32_t kv_heads, int32_t dim, int32_t dtype, int32_t cache_dtype,
                                 const float* k_scale, const float* v_scale, float scale, int32_t window, void* out,
                                 int64_t out_stride_t, int64_t out_stride_h, float* lse_out, void* workspace, size_t workspace_bytes,
                                 int32_t num_chunks, int32_t heads_per_group, int32_t rows_per_group,
                                 const uint64_t* visible, int64_t visible_stride, int32_t words, hipStream_t stream) {
  MLA_REQUIRE(q && k_cache && v_cache && block_table && seq_lens && out, MLA_ERR_NULL, "%s: null pointer argument", me);
  MLA_REQUIRE(!kTree || visible, MLA_ERR_NULL, "%s: null pointer argument", me);
  MLA_REQUIRE(!kTree || (words >= 1 && words <= kMostWords && max_q_len <= 64 * words && (num_tokens <= 1 || visible_stride >= words) && (uintptr_t)visible % 8 == 0), MLA_ERR_SHAPE,
              "%s: %d words of 64 bits for %d tokens (1 to %d words), rows %lld apart", me, words, max_q_len, kMostWords, (long long)visible_stride);
  MLA_REQUIRE((dtype == 0 || dtype == 2) && (cache_dtype == dtype || cache_dtype == 3), MLA_ERR_UNSUPPORTED,
              "%s: queries bf16 (0) or fp16 (2), caches of their type or e4m3 (3)", me);
  MLA_REQUIRE(dim == 64 || dim == 128 || dim == 256, MLA_ERR_UNSUPPORTED, "%s: heads of %d values (64, 128 or 256)", me, dim);
  MLA_REQUIRE(batch >= 0 && batch <= 65535 && max_q_len >= 1 && kv_heads >= 1 && q_heads >= kv_heads && q_heads % kv_heads == 0 && num_pages >= 1 &&
                  num_tokens >= 0 && num_chunks >= 0 && window >= 0 && max_blocks >= 1 && bt_stride >= max_blocks && (int64_t)max_q_len * q_heads < (1 << 24),
              MLA_ERR_SHAPE, "%s: batch %d, %d tokens each, %d query and %d key heads, %lld pages, %d chunks, window %d", me, batch, max_q_len,
              q_heads, kv_heads, (long long)num_pages, num_chunks, window);
  MLA_REQUIRE(page_size >= 16 && page_size % 16 == 0 && (int64_t)max_blocks * page_size <= (1 << 30), MLA_ERR_SHAPE,
              "%s: %d pages of %d tokens a request (pages of a multiple of 16, at most 2^30 tokens)", me, max_blocks, page_size);
  MLA_REQUIRE((int64_t)batch * max_blocks * page_size < (1ll << 35) && num_chunks < (1 << 24), MLA_ERR_SHAPE,
              "%s: %d requests of up to %lld tokens in %d chunks are more than the plan counts", me, batch, (long long)max_blocks * page_size, num_chunks);
  MLA_REQUIRE(query_start_loc || (int64_t)batch * max_q_len <= 0x7fffffff, MLA_ERR_SHAPE, "%s: %d requests of %d tokens: more than 2^31 - 1 rows", me,
              batch, max_q_len);
  const int es = cache_dtype == 3 ? 1 : 2, unit = 16 / es;
  const int64_t c_strides = kc_page_stride | kc_row_stride | kc_head_stride | vc_page_stride | vc_row_stride | vc_head_stride;
  MLA_REQUIRE((q_stride_t | q_stride_h) % 8 == 0 && c_strides % unit == 0 && (out_stride_t | out_stride_h) % 4 == 0 &&
                  !(((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) && !((uintptr_t)out & 7) && kc_row_stride >= 0 &&
                  vc_row_stride >= 0 && kc_row_stride * es * page_size < (1ll << 30) && vc_row_stride * es * page_size < (1ll << 30),
              MLA_ERR_SHAPE, "%s: heads must be 16-byte aligned (results: 8), the rows of a page within 1 GiB", me);
  if (batch == 0 || num_tokens == 0) return MLA_OK;
  Params p{};
  p.q = (const char*)q; p.q_st = q_stride_t * 2; p.q_sh = q_stride_h * 2;
  p.k = (const char*)k_cache; p.k_sp = kc_page_stride * es; p.k_sr = (int32_t)kc_row_stride * es; p.k_sh = kc_head_stride * es;
  p.v = (const char*)v_cache; p.v_sp = vc_page_stride * es; p.v_sr = (int32_t)vc_row_stride * es; p.v_sh = vc_head_stride * es;
  p.k_scale = k_scale; p.v_scale = v_scale;
  p.block_table = block_table; p.bt_stride = bt_stride; p.max_blocks = max_blocks;
  p.seq_lens = seq_lens; p.qsl = query_start_loc;
  p.num_tokens = num_tokens; p.num_pages = (int32_t)(num_pages < 0x7fffffff ? num_pages : 0x7fffffff);
  p.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz(page_size) : -1;
  p.page_size = page_size; p.batch = batch; p.max_q_len = max_q_len; p.kv_heads = kv_heads; p.group = q_heads / kv_heads;
  // (a window that no request outgrows is none; below it, window and tokens together stay within 32 bits)
  p.window = window < max_blocks * page_size ? window : 0; p.num_chunks = num_chunks;
  p.visible = visible; p.visible_stride = visible_stride; p.words = words;
  p.scale_log2 = scale * kLog2e;
  p.out = (char*)out; p.o_st = out_stride_t * 2; p.o_sh = out_stride_h * 2; p.lse = lse_out;
  const bool wide = kTree && rows_per_group == 128;
  MLA_REQUIRE(rows_per_group == 16 || rows_per_group == 32 || (rows_per_group == 64 && dim < 256) || wide, MLA_ERR_SHAPE,
              "%s: %d rows to a workgroup (16, 32, 64 of heads of up to 128%s)", me, rows_per_group, kTree ? ", 128" : "");
  MLA_REQUIRE(!wide || heads_per_group == 1, MLA_ERR_SHAPE, "%s: %d key heads to a workgroup of %d rows", me, heads_per_group, rows_per_group);
  const int rows = max_q_len * p.group, mt = rows_per_group / 16, waves = few_waves(rows_per_group, dim, es) ? 4 : 8;
  MLA_REQUIRE(heads_per_group >= 1 && heads_per_group <= waves && (heads_per_group & (heads_per_group - 1)) == 0 && kv_heads % heads_per_group == 0,
              MLA_ERR_SHAPE, "%s: %d of %d key heads to a workgroup of %d wavefronts (a power of two that divides both)", me, heads_per_group,
              kv_heads, waves);
  const int shift = __builtin_ctz(heads_per_group);
  p.heads_shift = shift;
  p.head_groups = kv_heads >> shift;
  // (a piece's start and join take about 3.5 us, a CU 26 KB per us)
  p.spare_units = (int32_t)(3.5f * 26e3f / (float)((int64_t)heads_per_group * 2 * dim * es * kUnit));
  const int row_groups = (rows + 16 * mt - 1) / (16 * mt);
  MLA_REQUIRE((int64_t)p.head_groups * row_groups <= 65535, MLA_ERR_SHAPE, "%s: %d head groups x %d row groups", me, p.head_groups, row_groups);
  const unsigned x = (unsigned)(num_chunks > 0 ? num_chunks : batch);
  MLA_REQUIRE((int64_t)x * waves * 64 < (1ll << 32), MLA_ERR_SHAPE, "%s: %d chunks are more than a launch takes", me, num_chunks);
  // (last: a caller that keeps scratch memory asks for it when all else has been found right)
  const size_t need = workspace_need(batch, max_q_len, q_heads, dim, num_chunks);
  MLA_REQUIRE(num_chunks == 0 || (workspace && (uintptr_t)workspace % 16 == 0 && workspace_bytes >= need), MLA_ERR_WORKSPACE,
              "%s: workspace of %zu bytes, %zu are needed", me, workspace ? workspace_bytes : 0, need);
  if (num_chunks > 0) {
    char* ws = (char*)workspace;
    const int64_t n = slots(batch, num_chunks) * max_q_len * q_heads;
    p.seg_ids = (int32_t*)ws;
    p.part_lse = (f32x2*)(ws + align256((int64_t)batch * 8));
    p.part_acc = (float*)((char*)p.part_lse + align256(n * 8));
  }
  if (wide) return launch_wide_rows(me, p, dtype, dim, cache_dtype == 3, x, stream);
  return dtype == 0 ? pick<kTree, __bf16>(me, p, dim, cache_dtype == 3, mt, row_groups, x, stream)
                    : pick<kTree, _Float16>(me, p, dim, cache_dtype == 3, mt, row_groups, x, stream);
}

}  // namespace gqa
}  // namespace mlahip
