// The rows of an accepted path moved to the places behind the context, in all layers' caches at once, when it is known which of a step's drafted tokens stay.
//
//   row(c + d) = row(c + accepted[d])   for d < kept, every cache of the list and every request b; its new length is c + kept
//   row(x): the cache row of a request's place x by its block table;  kept: how many of the first num_accepted entries are each larger than the one
//   before it, places of the request (c + accepted[d] < seq_lens[b]), and in pages that there are
// A path goes down a tree whose tokens stand behind their parents, so accepted[d] >= d, and a row that is overwritten is no later one's source.
//
// What bounds it: few rows of each request, read and written once, behind two dependent reads (the path, its pages).  A wavefront looks a request's path up,
// an entry to a lane, and moves 64 granules of its rows in one cache: as many rows at once as their granules leave lanes for.  A row is read in front of its
// own write; rows that are read later lie behind all places that have been written by then.
// us: 64 requests x 54 caches of 1024 and 128 bytes, 4 rows of 5 (8 MB read and written) 5.4; 256 requests x 64 caches x 4 rows of 2 KB (270 MB) 58, 4.6 TB/s.
// By a lane that looked its request's path up for itself 8.1 and 117; a wavefront for four caches one after the other, the path looked up once, 5.4 and 68
// (one takes up what another waits for); pieces of a row in neighbouring wavefronts 5.3 and 59.
#include "mla_common.hpp"
#include "../../include/mla_hip.h"
#include <string.h>

namespace mlahip {
namespace keep {

// (an address that comes as numbers is said to be in global memory: flat accesses wait for the LDS as well)
#define GLOBAL __attribute__((address_space(1)))

struct Cache { char* base; int64_t page_stride; uint32_t row_bytes, row_stride; };
constexpr int kCaches = 144;                                 // of a launch
struct Params {
  Cache caches[kCaches];
  const int32_t* table; int64_t table_stride; int32_t cols, page_size, page_shift, num_pages;
  const int32_t *context, *lens, *accepted, *num; int64_t accepted_stride; int32_t most;
  int32_t* kept;                                             // or null
  int32_t batch;
};
typedef const __attribute__((address_space(4))) int32_t* ConstPtr;

// kNt: past the caches.  Launches of 128 MB or more, every path counted as a whole one, go there: 270 MB moved 58 us, 62.5 through the caches; 77 MB at
// most 21.7 and 20.0; 8 MB 6.6 and 5.4.
template <typename V, bool kNt>
__global__ __launch_bounds__(256) void keep_rows_kernel(const Params p) {
  struct Move { int32_t from_page, from_row, to_page, to_row; };
  __shared__ Move list[4][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int b = blockIdx.x * 4 + wave;
  if (b >= p.batch) return;
  const int ctx = ((ConstPtr)p.context)[b], len = ((ConstPtr)p.lens)[b], num = ((ConstPtr)p.num)[b];
  const int n = ctx < 0 || num < 0 ? 0 : num < p.most ? num : p.most;
  Move* moves = list[wave];
  int last = -1, kept = 0;
  for (int d0 = 0; d0 < p.most; d0 += 64) {                  // (the first entries asked for together with the numbers above)
    const int d = d0 + lane;
    const int from = d < p.most ? p.accepted[b * p.accepted_stride + d] : -1;
    if (d0 >= n) break;
    int before = __builtin_amdgcn_update_dpp(last, from, 0x138, 0xf, 0xf, false);   // (of the lane below; the first one's: the last of the 64 before)
    struct Place { int32_t page, row; };
    auto place = [&](int64_t x) {
      if (x >= (int64_t)p.cols * p.page_size) return Place{-1, 0};
      const uint32_t at = (uint32_t)x, pi = p.page_shift >= 0 ? at >> p.page_shift : at / (uint32_t)p.page_size;
      return Place{p.table[b * p.table_stride + pi], (int32_t)(at - pi * (uint32_t)p.page_size)};
    };
    Place src{-1, 0}, dst{-1, 0};
    const bool inside = d < n && from > before && (int64_t)ctx + from < len;
    if (inside) {
      src = place((int64_t)ctx + from);
      dst = place((int64_t)ctx + d);
    }
    const bool good = inside && src.page >= 0 && src.page < p.num_pages && dst.page >= 0 && dst.page < p.num_pages;
    const uint64_t bad = ~__builtin_amdgcn_ballot_w64(good);
    const int run = bad ? __builtin_ctzll(bad) : 64;         // entries up to the first that ends the path
    kept += run;
    const bool moved = lane < run && from != d;
    const uint64_t all = __builtin_amdgcn_ballot_w64(moved);
    const int count = __builtin_popcountll(all);
    if (moved) moves[__builtin_popcountll(all & ((1ull << lane) - 1))] = Move{src.page, src.row, dst.page, dst.row};
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const Cache c = p.caches[blockIdx.y];
    const uint32_t granules = c.row_bytes / sizeof(V);
    const int shift = granules > 32 ? 6 : granules > 1 ? 32 - __builtin_clz(granules - 1) : 0, rows = 64 >> shift;
    const uint32_t at = (blockIdx.z << shift) + (lane & ((1 << shift) - 1));
    GLOBAL char* column = (GLOBAL char*)c.base + (int64_t)at * sizeof(V);
    auto spot = [&](int32_t page, int32_t row) { return (GLOBAL V*)(column + (page * c.page_stride + (int64_t)row * c.row_stride)); };
    constexpr int kAtOnce = 4;
    for (int m0 = at < granules ? lane >> shift : count; m0 < count; m0 += rows * kAtOnce) {
      V v[kAtOnce];
#pragma unroll
      for (int k = 0; k < kAtOnce; k++) {
        const int m = m0 + k * rows;
        if (m >= count) continue;
        const GLOBAL V* x = spot(moves[m].from_page, moves[m].from_row);
        if constexpr (kNt) v[k] = __builtin_nontemporal_load(x);
        else v[k] = *x;
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; k++) {
        const int m = m0 + k * rows;
        if (m >= count) continue;
        GLOBAL V* x = spot(moves[m].to_page, moves[m].to_row);
        if constexpr (kNt) __builtin_nontemporal_store(v[k], x);
        else *x = v[k];
      }
    }
    if (run < 64) break;
    last = __builtin_amdgcn_readlane(from, 63);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  if (p.kept && blockIdx.y == 0 && blockIdx.z == 0 && lane == 0) p.kept[b] = ctx < 0 ? ctx : ctx + kept;
}

}  // namespace keep
}  // namespace mlahip
using namespace mlahip;

extern "C" int mlahip_keep_rows(const mlahip_page_cache* caches, int32_t num_caches, int64_t num_pages, int32_t page_size, const int32_t* block_table,
                                int64_t bt_stride, int32_t max_blocks, const int32_t* context_lens, const int32_t* seq_lens, int32_t batch,
                                const int32_t* accepted, int64_t accepted_stride, int32_t max_accepted, const int32_t* num_accepted,
                                int32_t* kept_lens, hipStream_t stream) {
  const char* me = "mlahip_keep_rows";
  MLA_REQUIRE(num_caches >= 1 && num_pages >= 1 && num_pages <= 0x7fffffff && page_size >= 1 && max_blocks >= 1 && batch >= 0 && batch < (1 << 24) &&
                  (batch <= 1 || (bt_stride >= max_blocks && accepted_stride >= max_accepted)) && max_accepted >= 0,
              MLA_ERR_SHAPE, "%s: %d caches of %lld pages of %d, %d requests of %d pages, paths of %d", me, num_caches, (long long)num_pages, page_size, batch,
              max_blocks, max_accepted);
  MLA_REQUIRE(caches && (batch == 0 || (block_table && context_lens && seq_lens && num_accepted && kept_lens && (accepted || max_accepted == 0))), MLA_ERR_NULL,
              "%s: null pointer argument", me);
  for (int32_t i = 0; i < num_caches; i++) {
    const mlahip_page_cache& c = caches[i];
    MLA_REQUIRE(c.base, MLA_ERR_NULL, "%s: null pointer argument (cache %d)", me, i);
    MLA_REQUIRE(c.row_bytes >= 1 && c.row_stride_bytes >= c.row_bytes && c.row_stride_bytes < (1ll << 32) && c.row_bytes * page_size < (1ll << 31) &&
                    c.row_bytes <= (1 << 21) && c.page_stride_bytes >= c.row_bytes,
                MLA_ERR_SHAPE, "%s: cache %d: rows of %lld bytes, %lld apart, pages %lld apart", me, i, (long long)c.row_bytes,
                (long long)c.row_stride_bytes, (long long)c.page_stride_bytes);
    // rows inside pages, or pages inside rows
    MLA_REQUIRE(num_pages == 1 || (page_size - 1) * c.row_stride_bytes + c.row_bytes <= c.page_stride_bytes ||
                    (c.page_stride_bytes < c.row_stride_bytes && (num_pages - 1) * c.page_stride_bytes + c.row_bytes <= c.row_stride_bytes),
                MLA_ERR_SHAPE, "%s: cache %d: pages that share memory: rows of %lld bytes, %lld apart, %d to a page, pages %lld apart", me, i,
                (long long)c.row_bytes, (long long)c.row_stride_bytes, page_size, (long long)c.page_stride_bytes);
  }
  // Two moves of the same rows would take each other's results for what they read.  (A bit for an address: looked at again where two have one.)
  uint64_t bits[64] = {};
  for (int32_t i = 0; i < num_caches; i++) {
    const uint32_t at = (uint32_t)((uint64_t)(uintptr_t)caches[i].base * 0x9e3779b97f4a7c15ull >> 52);
    const bool met = bits[at >> 6] >> (at & 63) & 1;
    for (int32_t k = 0; met && k < i; k++)
      MLA_REQUIRE(caches[k].base != caches[i].base, MLA_ERR_UNSUPPORTED, "%s: caches %d and %d are the same", me, k, i);
    bits[at >> 6] |= 1ull << (at & 63);
  }
  if (batch == 0) return MLA_OK;
  const char *out = (const char*)kept_lens, *out_end = out + batch * 4ll;
  const auto meets = [&](const void* at, int64_t bytes) { return at && (const char*)at < out_end && out < (const char*)at + bytes; };
  MLA_REQUIRE(!meets(context_lens, batch * 4ll) && !meets(seq_lens, batch * 4ll) && !meets(num_accepted, batch * 4ll) &&
                  !meets(accepted, ((batch - 1) * accepted_stride + max_accepted) * 4) && !meets(block_table, ((batch - 1) * bt_stride + max_blocks) * 4),
              MLA_ERR_UNSUPPORTED, "%s: kept_lens shares memory with what is read", me);
  const uintptr_t fours = (uintptr_t)block_table | (uintptr_t)context_lens | (uintptr_t)seq_lens | (uintptr_t)accepted | (uintptr_t)num_accepted | (uintptr_t)kept_lens;
  MLA_REQUIRE(!(fours & 3), MLA_ERR_SHAPE, "%s: unaligned pointers", me);
  keep::Params p;
  p.table = block_table; p.table_stride = bt_stride; p.cols = max_blocks; p.page_size = page_size;
  p.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz(page_size) : -1;
  p.num_pages = (int32_t)num_pages;
  p.context = context_lens; p.lens = seq_lens; p.accepted = accepted; p.num = num_accepted; p.accepted_stride = accepted_stride; p.most = max_accepted;
  p.kept = kept_lens; p.batch = batch;
  // launches of the caches of one unit (16, 4 or 1 bytes: what addresses, strides and rows are multiples of); the first one writes the lengths
  for (const int unit : {16, 4, 1}) {
    int32_t next = 0;
    while (next < num_caches) {
      int32_t m = 0;
      int64_t most = 1, total = 0;
      for (; next < num_caches && m < keep::kCaches; next++) {
        const mlahip_page_cache& c = caches[next];
        const uint64_t bits = (uint64_t)(uintptr_t)c.base | (uint64_t)c.page_stride_bytes | (uint64_t)c.row_stride_bytes | (uint64_t)c.row_bytes;
        if ((bits & 15 ? bits & 3 ? 1 : 4 : 16) != unit) continue;
        p.caches[m++] = keep::Cache{(char*)c.base, c.page_stride_bytes, (uint32_t)c.row_bytes, (uint32_t)c.row_stride_bytes};
        most = c.row_bytes / unit > most ? c.row_bytes / unit : most;
        total += c.row_bytes;
      }
      if (m == 0) break;
      const dim3 grid((unsigned)((batch + 3) / 4), (unsigned)m, (unsigned)((most + 63) / 64));
      if (unit == 16 && (double)total * batch * max_accepted >= 0x1p27) hipLaunchKernelGGL((keep::keep_rows_kernel<u32x4, true>), grid, dim3(256), 0, stream, p);
      else if (unit == 16) hipLaunchKernelGGL((keep::keep_rows_kernel<u32x4, false>), grid, dim3(256), 0, stream, p);
      else if (unit == 4) hipLaunchKernelGGL((keep::keep_rows_kernel<uint32_t, false>), grid, dim3(256), 0, stream, p);
      else hipLaunchKernelGGL((keep::keep_rows_kernel<uint8_t, false>), grid, dim3(256), 0, stream, p);
      if (int e = check_launch(me)) return e;
      p.kept = nullptr;
    }
  }
  return MLA_OK;
}
