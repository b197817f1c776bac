// Attention of a tree's tokens where a key head has many rows (token x query head of the group): 128 of them to a workgroup, which share its keys.
//
// The formulas, the plan's partial results and their join are gqa_split.hpp's.  There 64 rows are a wavefront's, which walks keys of its own: each group of
// rows reads all keys again, a workgroup's wavefronts are joined at its end, and a SIMD has one wavefront, which does its products and its exponentials in
// turn.  Here
//   workgroup    one key head, 32 rows to each of four wavefronts, two workgroups to a CU (one with heads of 256, whose sums alone are 128 registers of a
//                lane and whose tiles 128 KB); no joins inside it, as each wavefront has all keys for its rows
//   tile         32 keys and values in LDS, 16 bits whatever the cache holds (16-bit ones are copied there directly, three tiles ahead, 8-bit ones are
//                converted once, two ahead), four buffers of each, one barrier to a tile
//   products     S^T = K Q^T and O^T = V^T P^T of 32x32x16: a lane's 16 scores are of one row, and their probabilities lie as the second product wants them
//   pipeline     a turn works on three tiles: scores of one, exponentials of the next older, the older still's products with values; no product waits for
//                another's result or for an exponential of its own turn, and both units work at once
// The order inside a turn is written down (sched_barrier): left to the compiler, products and exponentials lie in blocks of their own.
//
// Both operands of the probabilities make 3 products where a rounded one takes 2.  us, rows of a workgroup 64 / here, 8 key heads of 128 where nothing else
// is said: 8 requests of 480 rows, 2000-16 000 keys 363 / 265; 16 of 256, 1000-4000 keys 128 / 98; 8 of 256, 4 heads of 64, 109 / 73;
// 4 heads of 256, 8 requests of 480 rows, 2000-16 000 keys (32 rows there) 719 / 303; but one of 240, 4096 keys 27.2 / 30.9, and 32 of 32, 303 / 342.  That is 880 TFLOP/s of matrix products, with the card at 1370 of its 1400 W (zeros for data,
// same instructions: 17 % less time).  Eight wavefronts and 256 rows to a workgroup: 2 % faster at the largest of these, 12 % slower on average; products
// of 16x16x32, sums by dot products or by a column of ones, values one tile behind, other orders in a turn: all within 3 % or slower.
#include <utility>

#include "gqa_split.hpp"

namespace mlahip {
namespace gqa {

template <typename T> struct Wider;
template <> struct Wider<__bf16> {
  static __device__ __forceinline__ f32x16 mm(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(Types<__bf16>::v8, a), __builtin_bit_cast(Types<__bf16>::v8, b), c, 0, 0, 0);
  }
};
template <> struct Wider<_Float16> {
  static __device__ __forceinline__ f32x16 mm(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(Types<_Float16>::v8, a), __builtin_bit_cast(Types<_Float16>::v8, b), c, 0, 0, 0);
  }
};

template <int D, bool kFp8> struct Wide {
  static constexpr int waves = 4, threads = waves * 64, rows = waves * 32, keys = 32;
  static constexpr int lag = 2;                                                  // tiles by which the values are behind the keys
  static constexpr int row_b = D * 2, tile_b = keys * row_b;                     // in LDS
  static constexpr int src_b = kFp8 ? D : 2 * D, src_gran = src_b / 16;          // in the cache
  static constexpr int keys_per_load = 64 / src_gran;                            // of a wavefront's load
  static constexpr int loads = keys > waves * keys_per_load ? keys / (waves * keys_per_load) : 1;   // of a thread, of keys and of values
  static constexpr int loaders = keys / (keys_per_load * loads);                 // wavefronts that load
  static constexpr int words_b = rows * kTreeTiles * 4;
  static constexpr int lds_b = 8 * tile_b + words_b + 64;                        // keys of four tiles, values of four
  // Position of granule c of a key's row: c ^ k_swz(key) or v_swz(key).  Sixteen keys' rows at one granule hit different banks, and four neighbouring keys'
  // values at four; values of keys eight apart lie alike, so that they are a constant apart.
  static __device__ __forceinline__ int k_swz(int key) { return row_b >= 256 ? key & 15 : key >> 1 & 7; }
  static __device__ __forceinline__ int v_swz(int key) { return row_b >= 256 ? (key & 3) << 2 | (key >> 2 & 1) : (key >> 1 & 1) << 2 | (key >> 2 & 1) << 1; }
};

// A value that is worked out here and not where it is used, in front of what follows: the compiler would move it out of the block.
template <typename V> __device__ __forceinline__ V here(V x) {
  asm volatile("" : "+v"(x));
  return x;
}
__device__ __forceinline__ u32x2 read_tr(uint32_t lds_addr) {
  typedef __attribute__((__vector_size__(4 * sizeof(__bf16)))) __bf16 v4;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4bf16((LDS_PTR(v4))lds_addr));
}
template <typename T> __device__ __forceinline__ uint32_t times(uint32_t x, float f) {
  const typename Types<T>::v2 v = __builtin_bit_cast(typename Types<T>::v2, x);
  return __builtin_bit_cast(uint32_t, typename Types<T>::v2{(T)((float)v[0] * f), (T)((float)v[1] * f)});
}
template <int n> __device__ __forceinline__ void wait_loads() {
  static_assert(n <= 4 || n == 8, "the loads of a set");
  if constexpr (n == 0) MLA_WAIT_VMCNT(0);
  else if constexpr (n == 1) MLA_WAIT_VMCNT(1);
  else if constexpr (n == 2) MLA_WAIT_VMCNT(2);
  else if constexpr (n == 3) MLA_WAIT_VMCNT(3);
  else if constexpr (n == 4) MLA_WAIT_VMCNT(4);
  else MLA_WAIT_VMCNT(8);
}
template <int n> using Int = std::integral_constant<int, n>;
template <typename F, int... i> __device__ __forceinline__ void each_of(F f, std::integer_sequence<int, i...>) { (f(Int<i>{}), ...); }
template <int n, typename F> __device__ __forceinline__ void each(F f) { each_of(f, std::make_integer_sequence<int, n>{}); }
constexpr float kFine = 0x1p10f;                             // (log2 units: scores and references below it are off by half a step, 2^-15, at most)
constexpr float kNone = -0x1.fffffep127f, kAlways = -0x1p126f;   // limits of scores against a reference: of a row that has none, of one that is looked at in each tile
constexpr int kNowhere = 0x7effffc0;                         // a key that no request has (they have at most 2^30, and 2^24 tokens in front of the first)

template <typename T, int D, bool kFp8>
__global__ __launch_bounds__((Wide<D, kFp8>::threads), (D > 128 ? 1 : 2)) void gqa_tree_wide_kernel(const Params p, const int row_groups) {
  typedef Wide<D, kFp8> W;
  typedef Types<T> Ty;
  typedef Wider<T> Wd;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  uint32_t* tree_words = (uint32_t*)(lds + 8 * W::tile_b);   // [token][tile]
  int* flags = (int*)(lds + 8 * W::tile_b + W::words_b);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int l32 = lane & 31, h32 = lane >> 5;
  // Workgroups go to the eight XCDs in turn: the row groups of a piece, which read the same keys, eight apart.
  const int at8 = (int)blockIdx.x / (8 * row_groups), of8 = (int)blockIdx.x - at8 * 8 * row_groups, rg = of8 >> 3;
  const int unit_id = at8 * 8 + (of8 & 7), chunk = unit_id / p.kv_heads, head = unit_id - chunk * p.kv_heads;
  if (chunk >= (p.num_chunks > 0 ? p.num_chunks : p.batch)) return;
  const int row0 = rg * W::rows;
  auto units_of = [&](const Seq& s) {
    const int n = (s.len + W::keys - 1) / W::keys - first_key(p, s.key_0) / W::keys;
    return n > 0 ? n : 1;
  };

  // ---- which units are mine ----
  int v_cur = 0, v_end = 0, b = chunk, v_seq = 0;
  if (p.num_chunks > 0) {
    int tot = 0;
    for (int i = lane; i < p.batch; i += 64) tot += units_of(seq_of<true>(p, i));
    tot = __builtin_amdgcn_readlane(wave_incl_scan_dpp(tot), 63);
    const int size = __builtin_amdgcn_readfirstlane(chunk_units(tot, p.num_chunks));
    v_cur = chunk * size;
    v_end = v_cur + size < tot ? v_cur + size : tot;
    if (v_cur >= tot) return;
    int carry = 0;
    b = 0;
    for (int base = 0; base < p.batch; base += 64) {
      const int i = base + lane;
      const int run = wave_incl_scan_dpp(i < p.batch ? units_of(seq_of<true>(p, i)) : 0) + carry;
      const int n = __builtin_popcountll(__builtin_amdgcn_ballot_w64(i < p.batch && run <= v_cur));
      if (n > 0) v_seq = __builtin_amdgcn_readlane(run, n - 1);
      b += n;
      carry = __builtin_amdgcn_readlane(run, 63);
    }
  }

  const int lk = lane / W::src_gran, lp = lane % W::src_gran;
  // (16 bits: copies into LDS, where a lane's place is its number's: it fetches the granule that belongs there)
  const int k_swz = W::k_swz(wave * W::keys_per_load + lk), v_swz = W::v_swz(wave * W::keys_per_load + lk);
  const int k_off = lk * p.k_sr + (kFp8 ? lp : lp ^ k_swz) * 16, v_off = lk * p.v_sr + (kFp8 ? lp : lp ^ v_swz) * 16;
  const int k_off8 = lk * p.k_sr + (lp ^ k_swz ^ 8) * 16;     // (of keys eight further, where a load is that far from the one before)
  do {
    if (b >= p.batch) break;
    const Seq sq = seq_at<true>(p, b);
    const int units = units_of(sq);
    int u0 = 0, u1 = units;
    bool whole = true;
    if (p.num_chunks > 0) {
      u0 = v_cur - v_seq;
      u1 = v_end - v_seq < units ? v_end - v_seq : units;
      v_seq += units;
      v_cur = v_seq < v_end ? v_seq : v_end;
      whole = u0 == 0 && u1 == units;
      if (head == 0 && rg == 0 && threadIdx.x == 0) {
        GLOBAL int32_t* ids = (GLOBAL int32_t*)reload()->seg_ids + 2 * b;
        if (u0 == 0) ids[0] = whole ? -1 : chunk + b;
        if (u1 == units && !whole) ids[1] = chunk + b;
      }
    }
    const int rows = sq.s * p.group;
    if (row0 < rows) {
      const int unit0 = first_key(p, sq.key_0) / W::keys;
      const int key0 = (unit0 + u0) * W::keys, key_end = (unit0 + u1) * W::keys, key1 = key_end < sq.len ? key_end : sq.len;
      const int tiles = key1 > key0 ? (key1 - key0 + W::keys - 1) / W::keys : 0;

      // ---- where keys lie: page numbers of the wavefront's next 64 pages, one to a lane ----
      int have0 = 0, have = 0;
      auto pages_from = [&](int pi) {
        const int at = pi + lane;
        have0 = pi;
        const int page = p.block_table[(int64_t)b * p.bt_stride + (at < p.max_blocks ? at : p.max_blocks - 1)];
        have = page < 0 ? 0 : page < p.num_pages ? page : p.num_pages - 1;
      };
      auto page_of = [&](int key) { return __builtin_amdgcn_readfirstlane(p.page_shift >= 0 ? key >> p.page_shift : (int)((uint32_t)key / (uint32_t)p.page_size)); };
      const ParamsPtr first = reload();
      const char *k_head = p.k + (int64_t)head * first->k_sh, *v_head = p.v + (int64_t)head * first->v_sh;
      const bool one_page = (p.page_size & (W::keys - 1)) == 0;   // (a tile lies in one)
      // Set i: tile i's keys and tile i - lag's values, which meet the same turns.
      u32x4 in_k[W::loads], in_v[W::loads];                  // (8 bits: on their way to be converted)
      int64_t k_at[W::loads], v_at[W::lag + 1][W::loads];    // where a wavefront's loads begin: this tile's keys, its and the ones before it's values
      const bool alike = p.k_sp == p.v_sp && p.k_sr == p.v_sr;
      constexpr int kApart = W::keys / W::loads;             // keys between a wavefront's loads
      auto places = [&](int tile) {
        const int key = key0 + tile * W::keys + wave * W::keys_per_load;
#pragma unroll
        for (int j = 0; j < W::loads; j++) {
#pragma unroll
          for (int n = W::lag; n > 0; n--) v_at[n][j] = v_at[n - 1][j];
          if (j == 0 || !one_page) {
            const int pi = page_of(key + j * kApart);
            if ((uint32_t)(pi - have0) > 63u) pages_from(pi);
            const int page = __builtin_amdgcn_readlane(have, pi - have0), row = key + j * kApart - pi * p.page_size;
            k_at[j] = page * p.k_sp + row * p.k_sr;          // (a page's rows: below 2^30 bytes)
            v_at[0][j] = alike ? k_at[j] : page * p.v_sp + row * p.v_sr;
          } else {
            k_at[j] = k_at[0] + j * kApart * p.k_sr;
            v_at[0][j] = v_at[0][0] + j * kApart * p.v_sr;
          }
        }
      };
      const bool loader = wave < W::loaders;
      auto lds_place = [&](int buffer, int j) { return lds + buffer * W::tile_b + (wave * W::keys_per_load + j * kApart) * W::row_b; };
      const uint32_t lds_wave = __builtin_amdgcn_readfirstlane(lds_addr_of(lds) + wave * W::keys_per_load * W::row_b);
      const int sets = tiles > 0 ? tiles + W::lag : 0;
      auto ask = [&](int i) {
        if (!loader || i >= sets) return;
        places(i);
        auto load = [&](const char* from, int lane_offset) {
          return load_nt(__builtin_amdgcn_make_buffer_rsrc((void*)from, 0, 0x7fffffff, 0x00027000), lane_offset, 0);
        };
        const uint32_t k_to = lds_wave + (i & 3) * W::tile_b, v_to = lds_wave + (4 + (i - W::lag & 3)) * W::tile_b;
        if (i < tiles) {
#pragma unroll
          for (int j = 0; j < W::loads; j++) {
            if constexpr (kFp8) in_k[j] = load(k_head + k_at[j], k_off);
            else dma16_sv_m0add(k_head + k_at[j], kApart % 16 * j % 16 ? k_off8 : k_off, k_to, j * kApart * W::row_b);
          }
        }
        if (i >= W::lag) {
#pragma unroll
          for (int j = 0; j < W::loads; j++) {
            if constexpr (kFp8) in_v[j] = load(v_head + v_at[W::lag][j], v_off);
            else dma16_sv_m0add(v_head + v_at[W::lag][j], v_off, v_to, j * kApart * W::row_b);
          }
        }
      };
      pages_from(page_of(key0));

      // ---- the rows' tokens, what they see ----
      const int row_end = row0 + W::rows < rows ? row0 + W::rows : rows;
      const int tok_first = (int)((uint32_t)row0 / (uint32_t)p.group), tok_last = (int)((uint32_t)(row_end - 1) / (uint32_t)p.group);
      const int tree_tile0 = sq.key_0 & ~31;
      auto visible_of = [&](int token) {
        const ParamsPtr at = reload();
        const int64_t t = (int64_t)sq.q0 + token;
        return (const GLOBAL uint64_t*)at->visible + (t >= 0 && t < at->num_tokens ? t : 0) * at->visible_stride;
      };
      auto window_left = [&](const GLOBAL uint64_t* row) {
        const int own = sq.len - sq.key_0;
        return p.window - bits_below(row, own < 64 * p.words ? own : 64 * p.words);
      };
      if (key1 > sq.key_0) {
        for (int it = threadIdx.x; it < (tok_last - tok_first + 1) * kTreeTiles; it += W::threads) {
          const int k = it / kTreeTiles, n = it - k * kTreeTiles;
          const GLOBAL uint64_t* row = visible_of(tok_first + k);
          tree_words[it] = tree_word([&](int w) { return row[w]; }, p.words, tree_tile0 + n * 32, sq.key_0, sq.len, p.window > 0 ? -window_left(row) : 0);
        }
      }
      if (threadIdx.x == 0) flags[0] = 0;
      auto tile_bits = [&](int token, int key) {             // of 32 keys, without the window's begin
        const int n = (key - tree_tile0) / 32;
        return key < tree_tile0 ? 0xffffffffu : n < kTreeTiles ? tree_words[(token - tok_first) * kTreeTiles + n] : 0u;
      };

      // ---- the query: row l32 of the wavefront's, eight dims a step; zeros in a row that does not exist ----
      u32x4 qf[D / 16];
      const int r = row0 + wave * 32 + l32, rr = r < rows ? r : row0;
      const int tok = (int)((uint32_t)rr / (uint32_t)p.group);
      {
        const int64_t t = (int64_t)sq.q0 + tok;
        const bool ok = r < rows && t >= 0 && t < first->num_tokens;
        const GLOBAL char* src = (const GLOBAL char*)first->q + (ok ? t : 0) * first->q_st + (int64_t)(head * p.group + (rr - tok * p.group)) * first->q_sh +
                                 here(h32) * 16;   // (here: not kept in front of the loop over the pieces)
#pragma unroll
        for (int s = 0; s < D / 16; s++) qf[s] = ok ? *(const GLOBAL u32x4*)(src + s * 32) : u32x4{0u, 0u, 0u, 0u};
      }
      int lo = 0;
      if (p.window > 0) {
        const int left = window_left(visible_of(tok));
        lo = sq.key_0 - (left > 0 ? left : 0);
      }
      float scale_log2 = first->scale_log2 * (kFp8 && first->k_scale ? ((const GLOBAL float*)first->k_scale)[head] : 1.f);
      const int all_hi = sq.key_0, all_lo = p.window > 0 ? sq.len - p.window : 0, any_lo = p.window > 0 ? sq.key_0 - p.window : 0;
      int only = -1;                                         // the token that a pass is for, where the piece is done token by token
      while (true) {
        const bool one = only >= 0 || tok_first == tok_last;
        const int the_one = only >= 0 ? only : tok_first;
        int one_lo = 0;
        if (one && p.window > 0) {
          const int left = window_left(visible_of(the_one));
          one_lo = sq.key_0 - (left > 0 ? left : 0);
        }
        uint32_t odd = 0;
        f32x16 acc[D / 32];
        float y[16];                                         // scores against the reference, log2 units
        u32x4 pf[2], pl[2];                                  // probabilities of 32 keys, 16 a product, in two operands
        float sum[2] = {0.f, 0.f}, ref = 0.f, limit = kNone;  // limit: above which a score sets the row's reference anew
#pragma unroll
        for (int d = 0; d < D / 32; d++)
#pragma unroll
          for (int e = 0; e < 16; e++) acc[d][e] = 0.f;
#pragma unroll
        for (int e = 0; e < 16; e++) y[e] = -INFINITY;
        pf[0] = pf[1] = pl[0] = pl[1] = u32x4{0u, 0u, 0u, 0u};
        auto is_partial = [&](int tile_key) { return tile_key + W::keys > all_hi || tile_key < all_lo; };
        // Set i has come: 8-bit ones go to LDS as two granules of 16 bits.  Values: keys that no row sees are cleared, a value that is not finite and is
        // seen by some rows only is noted.
        auto come = [&](int i) {
          if (!loader || i >= sets) return;
          const int tile_key = key0 + (i - W::lag) * W::keys;   // (the values')
          const bool clear = i >= W::lag && is_partial(tile_key);
          auto cleared = [&](u32x4 x, int j) {
            const int k = wave * W::keys_per_load + j * kApart + lk, key = tile_key + k;
            bool seen = key >= (one ? one_lo : any_lo) && key < sq.len;
            if (one) seen = seen && (tile_bits(the_one, tile_key) >> k & 1);
#pragma unroll
            for (int e = 0; e < 4; e++) {
              x[e] = seen ? x[e] : 0u;
              odd |= one ? 0u : kFp8 ? ((x[e] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u : ((x[e] & Ty::kExp) + Ty::kLow) & 0x80008000u;
            }
            return x;
          };
          if constexpr (kFp8) {
            auto put = [&](int buffer, int j, u32x4 x, int swz) {
              char* row = lds_place(buffer, j) + lk * W::row_b;
              u32x4 y0, y1;
#pragma unroll
              for (int e = 0; e < 2; e++) {
                y0[2 * e] = Ty::from_e4m3(x[e], false); y0[2 * e + 1] = Ty::from_e4m3(x[e], true);
                y1[2 * e] = Ty::from_e4m3(x[2 + e], false); y1[2 * e + 1] = Ty::from_e4m3(x[2 + e], true);
              }
              *(u32x4*)(row + (((2 * lp) ^ swz) << 4)) = y0;
              *(u32x4*)(row + (((2 * lp + 1) ^ swz) << 4)) = y1;
            };
#pragma unroll
            for (int j = 0; j < W::loads; j++) {
              if (clear) in_v[j] = cleared(in_v[j], j);
              if (i < tiles) put(i & 3, j, in_k[j], k_swz);
              if (i >= W::lag) put(4 + (i - W::lag & 3), j, in_v[j], v_swz);
            }
          } else if (clear) {
#pragma unroll
            for (int j = 0; j < W::loads; j++) {
              u32x4* at = (u32x4*)(lds_place(4 + (i - W::lag & 3), j) + lane * 16);
              *at = cleared(*at, j);
            }
          }
        };
        // All sets up to i are there, as far as the wavefront's own loads go; set i + 1 may still be under way.
        auto wait = [&](int i) {
          if constexpr (!kFp8) {
            const bool keys = i + 1 < tiles, values = i + 1 >= W::lag && i + 1 < sets;
            if (keys && values) wait_loads<2 * W::loads>();
            else if (keys || values) wait_loads<W::loads>();
            else wait_loads<0>();
          }
        };
        // Addresses in LDS of a lane's first granule of this tile's keys, and of the values of the one before it.  (A granule 2 n further: bits of n are
        // flipped.  Worked out in front of the loop, by the lane's number hidden from the compiler: it would keep them in memory until then.)
        uint32_t k_lane = 0, v_lane = 0;
        auto read_k = [&](int n) { return *(LDS_PTR(const u32x4))(k_lane ^ n << 5); };   // 16 dims
        auto read_v = [&](int n) {                           // 32 dims, 16 keys in the order of the scores: 4 h32 + 0 .. 3, then 8 further
          const uint32_t row = (v_lane ^ n % (D / 32) << 6) + n / (D / 32) * 16 * W::row_b;
          const u32x2 x0 = read_tr(row), x1 = read_tr(row + 8 * W::row_b);
          return u32x4{x0[0], x0[1], x1[0], x1[1]};
        };
        // Where a score outgrows its row's reference the wavefront's are set anew (all of them, the next would follow soon: fp16 6 % faster than one by one):
        // what is summed up, and the probabilities that are not yet, by a whole power of two.
        auto check = [&](int key, bool partial, float most) {
          if (partial) {
            const uint32_t bits = (tile_bits(tok, key) & ~bits_to(lo - key)) >> 4 * h32;
            most = -INFINITY;
#pragma unroll
            for (int e = 0; e < 16; e++) {
              y[e] = bits & 1u << ((e & 3) + 8 * (e >> 2)) ? y[e] : -INFINITY;
              most = fmaxf(most, y[e]);
            }
          }
          if (__builtin_expect(__builtin_amdgcn_ballot_w64(most > limit) != 0, 0)) {
            most = fmaxf(most, __shfl_xor(most, 32, 64));
            // Large scores: the turn's y is an unrounded score less the reference, the tile's that set the reference a rounded one's, and a reference
            // does not move by less than its own steps: equal scores would weigh more or less by the tile that they lie in (at 2^20 by 4 %, beyond 2^25 all of it).
            // So each tile of such a row is looked at here, and has its products again: rounded, then less the reference, which is a whole number near them.
            // (8 requests of 480 rows, 2000-16 000 keys 269 us, all rows such 428; every row's products rounded in the turn instead 2.5 % more for all.)
            const bool anew = most > -INFINITY, large = anew && (fabsf(ref) >= kFine || fabsf(ref + most) >= kFine);
            const float before = ref;
            if (__builtin_expect(__builtin_amdgcn_ballot_w64(large) != 0, 0)) {
              f32x16 sc = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int n = 0; n < D / 16; n++) sc = Wd::mm(read_k(n), qf[n], sc);
              float all = -INFINITY;
#pragma unroll
              for (int e = 0; e < 16; e++) {
                const float s = here(sc[e] * scale_log2);      // (by itself, not one operation with the difference)
                y[e] = large && y[e] != -INFINITY ? s : y[e];
                all = fmaxf(all, y[e]);
              }
              all = fmaxf(all, __shfl_xor(all, 32, 64));
              if (large) {
                most = all;
                ref = 0.f;
              }
            }
            if (anew) {
              float raise = __builtin_ceilf(most - (fabsf(ref + most) < 0x1p20f ? Ty::kBelow : 0.f));
              // (a row that has a reference keeps it or gets a higher one)
              raise = limit == kNone ? raise : fmaxf(raise, before - ref);
              const float f = limit == kNone ? 1.f : fast_exp2(before - (ref + raise));   // (zeros so far)
              ref += raise;
              limit = fabsf(ref) < kFine ? Ty::kBelow + Ty::kOutgrown : kAlways;
              sum[0] *= f;
              sum[1] *= f;
#pragma unroll
              for (int d = 0; d < D / 32; d++)
#pragma unroll
                for (int e = 0; e < 16; e++) acc[d][e] *= f;
#pragma unroll
              for (int e = 0; e < 16; e++) y[e] -= raise;
#pragma unroll
              for (int t = 0; t < 2; t++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                  pf[t][e] = times<T>(pf[t][e], f);
                  pl[t][e] = times<T>(pl[t][e], f);
                }
            }
          }
        };
        // One turn: the scores of the next 32 keys, these ones' probabilities, the products of the ones before with their values.  Products and the
        // rest take turns, in this order: the matrix cores work on the one while the wavefront issues the other.  D / 16 products for the scores, S, and
        // D / 16 operands of values, each with the probabilities' first and second ones, h and l:
        //   D / 64 times  S h S h S l S l, with three quarters of the probabilities, then  D / 64 times  h h l l, with the others and the new scores' maximum
        auto turn = [&] {
          constexpr int kBlocks = D / 64, kSlots = 12 * kBlocks, kA = 8 * kBlocks, kParts = kBlocks > 1 ? 2 : 1;
          const f32x16 zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
          f32x16 sc;
          u32x4 k[3], v[4], pn[2], ln[2];
          k[0] = read_k(0); k[1] = read_k(1);
          v[0] = read_v(0); v[1] = read_v(1);
          float x[16], most = -INFINITY;
          uint32_t w[8];
          auto exps = [&](int c) {                           // c: a pair of scores
#pragma unroll
            for (int e = 2 * c; e < 2 * c + 2; e++) x[e] = fast_exp2(here(y[e]));
            x[2 * c] = here(x[2 * c]);
            x[2 * c + 1] = here(x[2 * c + 1]);
          };
          auto add = [&](int c) {
            sum[0] = here(sum[0] + x[2 * c]);
            sum[1] = here(sum[1] + x[2 * c + 1]);
          };
          auto split = [&](int c) {                          // into the first operand and the rest
            add(c);
            w[c] = here(__builtin_bit_cast(uint32_t, typename Ty::v2{(T)x[2 * c], (T)x[2 * c + 1]}));
            const typename Ty::v2 first = __builtin_bit_cast(typename Ty::v2, w[c]);
#pragma unroll
            for (int e = 0; e < 2; e++) x[2 * c + e] = here(__builtin_fmaf(x[2 * c + e], kWhole, -(float)first[e]));
          };
          auto ends = [&](int c) {
            const uint32_t z = here(__builtin_bit_cast(uint32_t, typename Ty::v2{(T)x[2 * c], (T)x[2 * c + 1]}));
            pn[c >> 2][c & 3] = w[c];
            ln[c >> 2][c & 3] = z;
          };
          // pairs kFirst .. kFirst + n of the scores in kOf slots, one stage behind the other: what slot i does
          auto pairs = [&](auto i, auto kOf, auto kFirst, auto n) {
            each<n() + 2>([&](auto q) {
              if constexpr (q() * kOf() / (n() + 2) == i()) {
                if constexpr (q() < n()) exps(kFirst() + q());
                if constexpr (q() > 0 && q() <= n()) split(kFirst() + q() - 1);
                if constexpr (q() > 1) ends(kFirst() + q() - 2);
              }
            });
          };
          each<kSlots>([&](auto slot) {
            constexpr int i = slot();
            // reads: an operand of scores four slots in front of its product, of values as their places get free
            if constexpr (i < kA && i % 2 == 0 && i / 2 + 2 < D / 16) k[(i / 2 + 2) % 3] = read_k(i / 2 + 2);
            each<D / 16 - 2>([&](auto n2) {
              // (operand n - 4, whose place it takes, is behind its products, of which the second phase's come four slots apart and not eight)
              constexpr int n = n2() + 2, late = n - 2 * kBlocks;
              constexpr int at = late < 0 ? n / 2 * 8 + n % 2 * 2 - 5 : late < 2 ? kA - 7 + 2 * late : late < 4 ? kA - 6 + 2 * late : kA + late / 2 * 4 - 5 + late % 2;
              if constexpr (at == i) v[n % 4] = read_v(n);
            });
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (i < kA && i % 2 == 0) {
              sc = Wd::mm(k[i / 2 % 3], qf[i / 2], i == 0 ? zero : sc);
            } else {
              // operand n's first or second product
              constexpr int of4 = i < kA ? i / 2 % 4 : i % 4, n = (i < kA ? i / 8 : kBlocks + (i - kA) / 4) * 2 + of4 % 2, t = n / (D / 32), d = n % (D / 32);
              acc[d] = Wd::mm(v[n % 4], of4 < 2 ? pf[t] : pl[t], acc[d]);
            }
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (i < kA) {
              constexpr int kOf = kA / kParts;
              pairs(Int<i % kOf>{}, Int<kOf>{}, Int<i / kOf * (6 / kParts)>{}, Int<6 / kParts>{});
            } else {
              constexpr int kEach = 4 * kBlocks / kParts;
              pairs(Int<(i - kA) % kEach>{}, Int<kEach>{}, Int<6 + (i - kA) / kEach * (2 / kParts)>{}, Int<2 / kParts>{});
              constexpr int f = i - kA - 1, kOf = 4 * kBlocks - 1;
              if constexpr (f >= 0) {
#pragma unroll
                for (int e = 16 * f / kOf; e < 16 * (f + 1) / kOf; e++) y[e] = __builtin_fmaf(sc[e], scale_log2, -ref);
#pragma unroll
                for (int e = 16 * f / kOf; e < 16 * (f + 1) / kOf; e++) most = fmaxf(most, y[e]);
                most = here(most);
              }
            }
            __builtin_amdgcn_sched_barrier(0);
          });
#pragma unroll
          for (int t = 0; t < 2; t++) { pf[t] = pn[t]; pl[t] = ln[t]; }
          return most;
        };
        ask(0);
        lds_barrier();                                       // (the words and the flag are there; nobody reads the tiles of the pass before)
        for (int n = threadIdx.x; n < W::lag * W::tile_b / 16; n += W::threads) ((u32x4*)(lds + (8 - W::lag) * W::tile_b))[n] = u32x4{0u, 0u, 0u, 0u};
        // (the queries and the keys' scale have arrived here: the compiler would wait for them, and so for all loads, at the loop's top)
        asm volatile("" : "+v"(scale_log2));
#pragma unroll
        for (int s = 0; s < D / 16; s++) asm volatile("" : "+v"(qf[s]));
        if constexpr (kFp8) come(0);
        ask(1);
        if constexpr (!kFp8) wait(0);
        lds_barrier();
        if constexpr (!kFp8) ask(2);
        {
          int l = lane;
          asm volatile("" : "+v"(l));
          const int key = l & 31, value = 4 * (l >> 5) + (l >> 2 & 3);
          k_lane = lds_addr_of(lds) + key * W::row_b + (((l >> 5) ^ W::k_swz(key)) << 4);
          v_lane = lds_addr_of(lds) + (8 - W::lag) * W::tile_b + value * W::row_b + (((2 * (l >> 4 & 1) + (l >> 1 & 1)) ^ W::v_swz(value)) << 4) + (l & 1) * 8;
        }
        // Tile i's keys meet the values of the tile two before it (none: zeros); behind the last one, two tiles' values are left.
        for (int i = 0; i < sets; i++) {
          const int tile_key = i < tiles ? key0 + i * W::keys : kNowhere;
          const float most = turn();
          check(tile_key, i >= tiles || is_partial(tile_key), most);
          // set i + 1 comes, set i + 3 (8 bits: i + 2) is asked for
          wait(i + 1);
          come(i + 1);
          if constexpr (kFp8) ask(i + 2);
          lds_barrier();
          if constexpr (!kFp8) ask(i + 3);
          // (the next tile's: four buffers in turn)
          const int k_next = (i + 1 & 3) ? W::tile_b : -3 * W::tile_b, v_next = (i + 1 - W::lag & 3) ? W::tile_b : -3 * W::tile_b;
          k_lane += k_next;
          v_lane += v_next;
        }
        MLA_WAIT_VMCNT(0);

        // ---- done again, token by token? ----
        bool by_token = false;
        if (only < 0 && tok_first != tok_last) {
          if (odd) flags[0] = 1;
          lds_barrier();
          by_token = flags[0] != 0;
        }
        if (!by_token) {
          const ParamsPtr last = reload();
          // (waited for here: a wavefront that makes no use of it would take the load along, and the next piece's loop wait for it at its top)
          const float vs = here(kFp8 && last->v_scale ? ((const GLOBAL float*)last->v_scale)[head] : 1.f);
          const int64_t t = (int64_t)sq.q0 + tok;
          // (the sum is of the probabilities in fp32: both operands of one are kWhole of it up to their rounding)
          const float total = sum[0] + sum[1] + __shfl_xor(sum[0] + sum[1], 32, 64), inv = total == 0.f ? 0.f : vs / (total * kWhole);
          const f32x2 lse2 = total == 0.f ? f32x2{-INFINITY, 0.f} : lse_of(ref, fast_log2(total));
          if (r < rows && (only < 0 || tok == only) && (!whole || (t >= 0 && t < last->num_tokens))) {
            const int qh = head * p.group + (r - tok * p.group);
            if (whole) {
              if (last->lse && h32 == 0) ((GLOBAL float*)last->lse)[t * (p.kv_heads * p.group) + qh] = lse2[0] * kLn2;
              GLOBAL char* dst = (GLOBAL char*)last->out + t * last->o_st + (int64_t)qh * last->o_sh + here(h32) * 8;
#pragma unroll
              for (int d = 0; d < D / 32; d++)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                  typename Ty::v4 y;
#pragma unroll
                  for (int c = 0; c < 4; c++) y[c] = (T)(acc[d][e + c] * inv);
                  *(GLOBAL typename Ty::v4*)(dst + d * 64 + e * 4) = y;
                }
            } else {
              const int64_t slot = ((int64_t)(chunk + b) * p.kv_heads + head) * (p.max_q_len * p.group) + r;
              if (h32 == 0) ((GLOBAL f32x2*)last->part_lse)[slot] = lse2;
              GLOBAL float* dst = (GLOBAL float*)last->part_acc + slot * D + h32 * 4;
#pragma unroll
              for (int d = 0; d < D / 32; d++)
#pragma unroll
                for (int e = 0; e < 16; e += 4)
                  *(GLOBAL f32x4*)(dst + d * 32 + e * 2) = f32x4{acc[d][e] * inv, acc[d][e + 1] * inv, acc[d][e + 2] * inv, acc[d][e + 3] * inv};
            }
          }
        }
        if (by_token) only = tok_first;
        else if (only < 0 || ++only > tok_last) break;
      }
      lds_barrier();                                         // (the flag and the words have been read)
    }
    b++;
  } while (v_cur < v_end);
}

template <typename T, int D, bool kFp8>
int launch_wide(const char* me, const Params& p, unsigned x, hipStream_t st) {
  typedef Wide<D, kFp8> W;
  const int rc = ensure_dynamic_lds((const void*)gqa_tree_wide_kernel<T, D, kFp8>, W::lds_b, me);
  if (rc != MLA_OK) return rc;
  const int64_t row_groups = (p.max_q_len * p.group + W::rows - 1) / W::rows, units = ((int64_t)x * p.kv_heads + 7) / 8 * 8;
  MLA_REQUIRE(units * row_groups * W::threads < (1ll << 32), MLA_ERR_SHAPE, "%s: %u pieces of %d key heads in %lld groups of rows are more than a launch takes",
              me, x, p.kv_heads, (long long)row_groups);
  hipLaunchKernelGGL((gqa_tree_wide_kernel<T, D, kFp8>), dim3((unsigned)(units * row_groups)), dim3(W::threads), W::lds_b, st, p, (int)row_groups);
  if (int e = check_launch(me)) return e;
  return p.num_chunks > 0 ? launch_join<true, T, D>(me, p, st) : MLA_OK;
}

template <typename T>
int pick_wide(const char* me, const Params& p, int dim, bool fp8, unsigned x, hipStream_t st) {
  if (dim == 64) return fp8 ? launch_wide<T, 64, true>(me, p, x, st) : launch_wide<T, 64, false>(me, p, x, st);
  if (dim == 256) return fp8 ? launch_wide<T, 256, true>(me, p, x, st) : launch_wide<T, 256, false>(me, p, x, st);
  return fp8 ? launch_wide<T, 128, true>(me, p, x, st) : launch_wide<T, 128, false>(me, p, x, st);
}
int launch_wide_rows(const char* me, const Params& p, int dtype, int dim, bool fp8, unsigned x, hipStream_t st) {
  return dtype == 0 ? pick_wide<__bf16>(me, p, dim, fp8, x, st) : pick_wide<_Float16>(me, p, dim, fp8, x, st);
}

}  // namespace gqa
}  // namespace mlahip
