// Pages of a cache copied, forked (their filled rows only) or moved with the block table rewritten, in all layers' tensors at once.
//
//   cache[dst[i], r] = cache[src[i], r]   for r < rows[i], every cache of the list and every pair i
//   table entries that name a source name its destination afterwards
// The pairs are known on the host (the scheduler makes them) and travel as kernel arguments, with the caches' addresses: no copy of
// them to the GPU in front of the launch, and they are checked before it: a destination is named once and is no pair's source, so
// the order of the copies does not matter.  Where a table follows, a source is named once too: a page moves to one place.
//
// What bounds it is memory, each byte read and written once; a workgroup copies a piece of one pair's page in one cache.  A launch of 32 MB or
// more, filled rows counted as whole pages, goes past the caches, which would give up other lines for it, in pieces of 4 KB: together in flight they are neighbours in memory.  us
// through the caches / past them, pieces of 4 KB / 32 KB, behind 2 GB of other writes: 63 MB (7 pairs x 34 caches) 37 / 27, 42 / 29; 418 MB 170 / 140, 185 /
// 162; 2.5 GB 922 / 826, 1044 / 977.  Where the same pages are copied again and again, 47 MB 17.8 / 19.2, 105 MB 47 / 41, 2.5 GB 904 / 819 (6.1 TB/s read
// and written; a plain copy of 2 GiB 4.9).  Smaller launches go through the caches, in pieces of 8 KB: 12 MB 5.6, past them 9.9.
#include <stdlib.h>
#include <string.h>

#include "mla_common.hpp"
#include "../../include/mla_hip.h"

namespace mlahip {
namespace pages {

// (an address that comes as numbers is said to be in global memory: flat accesses wait for the LDS as well)
#define GLOBAL __attribute__((address_space(1)))

struct Cache { char* base; int64_t page_stride; uint32_t row_bytes, row_stride; };
// caches, then sources and destinations, then filled rows (a launch takes as many of either as fit)
constexpr int kArgBytes = 3840;
struct Params {
  uint32_t words[kArgBytes / 4];
  int32_t* table; int64_t table_stride; int32_t table_rows, table_cols;
  int32_t num_caches, num_pairs, page_size, part, piece;     // piece: 16-byte (or smaller) units of a workgroup
};

// kNt: past the caches (host: pieces of a unit to a thread)
template <typename V, bool kNt>
__global__ __launch_bounds__(256) void copy_pages_kernel(const Params p) {
  const uint32_t* pairs = p.words + p.num_caches * (int)(sizeof(Cache) / 4);
  const int pair = blockIdx.z;
  if (pair == p.num_pairs) {                                 // the table: an entry to a thread
    const int64_t n = (int64_t)p.table_rows * p.table_cols, step = (int64_t)gridDim.x * gridDim.y * 256;
    for (int64_t i = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 256 + threadIdx.x; i < n; i += step) {
      const int64_t r = i / p.table_cols;
      int32_t* at = p.table + r * p.table_stride + (i - r * p.table_cols);
      const int32_t page = *at;
      int32_t to = page;
      for (int k = 0; k < p.num_pairs; k++) to = page == (int32_t)pairs[2 * k] ? (int32_t)pairs[2 * k + 1] : to;
      if (to != page) *at = to;
    }
    return;
  }
  const uint32_t* words = p.words + blockIdx.y * (int)(sizeof(Cache) / 4);
  Cache c;
  c.base = (char*)((uint64_t)words[0] | (uint64_t)words[1] << 32);
  c.page_stride = (int64_t)((uint64_t)words[2] | (uint64_t)words[3] << 32);
  c.row_bytes = words[4];
  c.row_stride = words[5];
  const uint32_t rows = p.part ? pairs[2 * p.num_pairs + pair] : (uint32_t)p.page_size;
  const uint32_t row_units = c.row_bytes / sizeof(V), units = rows * row_units;
  const uint32_t begin = blockIdx.x * (uint32_t)p.piece, end = begin + p.piece < units ? begin + p.piece : units;
  const GLOBAL char* src = (const GLOBAL char*)c.base + (int64_t)(int32_t)pairs[2 * pair] * c.page_stride;
  GLOBAL char* dst = (GLOBAL char*)c.base + (int64_t)(int32_t)pairs[2 * pair + 1] * c.page_stride;
  if (c.row_bytes == c.row_stride) {
    uint32_t i = begin + threadIdx.x;
    if constexpr (kNt) {
      if (i < end) __builtin_nontemporal_store(__builtin_nontemporal_load((const GLOBAL V*)src + i), (GLOBAL V*)dst + i);
    } else {
      // (four loads on their way together: the compiler does not move one ahead of a store that might touch its bytes)
      for (; i + 768 < end; i += 1024) {
        V v[4];
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = ((const GLOBAL V*)src)[i + k * 256];
#pragma unroll
        for (int k = 0; k < 4; k++) ((GLOBAL V*)dst)[i + k * 256] = v[k];
      }
      for (; i < end; i += 256) ((GLOBAL V*)dst)[i] = ((const GLOBAL V*)src)[i];
    }
  } else {
    for (uint32_t i = begin + threadIdx.x; i < end; i += 256) {
      const uint32_t r = i / row_units;
      const uint64_t at = (uint64_t)r * c.row_stride + (i - r * row_units) * (uint32_t)sizeof(V);
      *(GLOBAL V*)(dst + at) = *(const GLOBAL V*)(src + at);
    }
  }
}

// A destination twice, or one that is a source too, or, where pages move, a source twice: what is wrong and the pair's number.
enum { kFine, kNoMemory, kDestination, kSource };
struct Clash { int what; int32_t pair; };
Clash clash(const int32_t* src, const int32_t* dst, int32_t n, int64_t num_pages, bool moves) {
  if (n <= 48) {
    for (int32_t i = 0; i < n; i++)
      for (int32_t k = 0; k < n; k++) {
        if ((k < i && dst[k] == dst[i]) || src[k] == dst[i]) return {kDestination, i};
        if (moves && k < i && src[k] == src[i]) return {kSource, i};
      }
    return {kFine, -1};
  }
  unsigned char* seen = (unsigned char*)calloc((size_t)num_pages, 1);
  if (!seen) return {kNoMemory, -1};
  Clash at{kFine, -1};
  for (int32_t i = 0; i < n; i++) {
    if (moves && seen[src[i]] && at.what == kFine) at = {kSource, i};
    seen[src[i]] = 1;
  }
  for (int32_t i = 0; i < n && at.what == kFine; i++) {
    if (seen[dst[i]]) at = {kDestination, i};
    seen[dst[i]] = 1;
  }
  free(seen);
  return at;
}

}  // namespace pages
}  // namespace mlahip
using namespace mlahip;

extern "C" int mlahip_copy_pages(const mlahip_page_cache* caches, int32_t num_caches, const int32_t* src, const int32_t* dst,
                                 const int32_t* rows, int32_t num_pairs, int64_t num_pages, int32_t page_size, int32_t* block_table,
                                 int64_t bt_stride, int32_t bt_rows, int32_t bt_cols, hipStream_t stream) {
  const char* me = "mlahip_copy_pages";
  MLA_REQUIRE(num_caches >= 1 && num_pairs >= 0 && num_pages >= 1 && num_pages <= 0x7fffffff && page_size >= 1, MLA_ERR_SHAPE,
              "%s: %d caches, %d pairs, %lld pages of %d", me, num_caches, num_pairs, (long long)num_pages, page_size);
  MLA_REQUIRE(caches && (num_pairs == 0 || (src && dst)), MLA_ERR_NULL, "%s: null pointer argument", me);
  MLA_REQUIRE(!block_table || (bt_rows >= 0 && bt_cols >= 0 && bt_stride >= bt_cols && (uintptr_t)block_table % 4 == 0), MLA_ERR_SHAPE,
              "%s: block table of %d x %d, stride %lld", me, bt_rows, bt_cols, (long long)bt_stride);
  MLA_REQUIRE(!(block_table && rows), MLA_ERR_UNSUPPORTED, "%s: a moved page is moved whole (no rows beside a block table)", me);
  for (int32_t i = 0; i < num_caches; i++) {
    const mlahip_page_cache& c = caches[i];
    MLA_REQUIRE(c.base, MLA_ERR_NULL, "%s: null pointer argument (cache %d)", me, i);
    MLA_REQUIRE(c.row_bytes >= 1 && c.row_stride_bytes >= c.row_bytes && c.row_stride_bytes < (1ll << 32) &&
                    c.row_bytes * page_size < (1ll << 31) && c.page_stride_bytes >= c.row_bytes,
                MLA_ERR_SHAPE, "%s: cache %d: rows of %lld bytes, %lld apart, pages %lld apart", me, i, (long long)c.row_bytes,
                (long long)c.row_stride_bytes, (long long)c.page_stride_bytes);
    // rows inside pages, or pages inside rows
    MLA_REQUIRE(num_pages == 1 || (page_size - 1) * c.row_stride_bytes + c.row_bytes <= c.page_stride_bytes ||
                    (c.page_stride_bytes < c.row_stride_bytes && (num_pages - 1) * c.page_stride_bytes + c.row_bytes <= c.row_stride_bytes),
                MLA_ERR_SHAPE, "%s: cache %d: pages that share memory: rows of %lld bytes, %lld apart, %d to a page, pages %lld apart", me, i,
                (long long)c.row_bytes, (long long)c.row_stride_bytes, page_size, (long long)c.page_stride_bytes);
  }
  for (int32_t i = 0; i < num_pairs; i++) {
    MLA_REQUIRE(src[i] >= 0 && src[i] < num_pages && dst[i] >= 0 && dst[i] < num_pages, MLA_ERR_SHAPE,
                "%s: pair %d copies page %d to %d of %lld", me, i, src[i], dst[i], (long long)num_pages);
    MLA_REQUIRE(!rows || (rows[i] >= 0 && rows[i] <= page_size), MLA_ERR_SHAPE, "%s: pair %d copies %d rows of %d", me, i,
                rows ? rows[i] : 0, page_size);
  }
  const pages::Clash bad = pages::clash(src, dst, num_pairs, num_pages, block_table != nullptr);
  MLA_REQUIRE(bad.what != pages::kNoMemory, MLA_ERR_WORKSPACE, "%s: no host memory for %lld marks", me, (long long)num_pages);
  MLA_REQUIRE(bad.what != pages::kDestination, MLA_ERR_UNSUPPORTED, "%s: page %d is written by pair %d and read or written by another", me,
              dst[bad.pair], bad.pair);
  MLA_REQUIRE(bad.what != pages::kSource, MLA_ERR_UNSUPPORTED, "%s: page %d moves to two places (again by pair %d)", me, src[bad.pair], bad.pair);
  if (num_pairs == 0) return MLA_OK;

  // A launch takes as many pairs and caches as its arguments hold, the caches of one unit (16, 4 or 1 bytes: what addresses, strides and
  // rows are multiples of).  A batch of pairs takes the table along in its first launch.
  constexpr int kCacheBytes = (int)sizeof(pages::Cache), kMostPairs = 192;
  constexpr uint64_t kPast = 32ull << 20;
  const int pair_bytes = rows ? 12 : 8;
  for (int32_t p0 = 0; p0 < num_pairs; p0 += kMostPairs) {
    const int32_t n = num_pairs - p0 < kMostPairs ? num_pairs - p0 : kMostPairs;
    bool table = block_table && bt_rows > 0 && bt_cols > 0;
    const int32_t room = (pages::kArgBytes - n * pair_bytes) / kCacheBytes;
    for (const int unit : {16, 4, 1}) {
      int32_t next = 0;
      while (next < num_caches) {
        pages::Params p;
        uint64_t most = 0, least = ~0ull, total = 0;
        int32_t m = 0;
        for (; next < num_caches && m < room; next++) {
          const mlahip_page_cache& c = caches[next];
          const uint64_t bits = (uint64_t)(uintptr_t)c.base | (uint64_t)c.page_stride_bytes | (uint64_t)c.row_stride_bytes | (uint64_t)c.row_bytes;
          if ((bits & 15 ? bits & 3 ? 1 : 4 : 16) != unit) continue;
          const pages::Cache to{(char*)c.base, c.page_stride_bytes, (uint32_t)c.row_bytes, (uint32_t)c.row_stride_bytes};
          memcpy(p.words + m * (kCacheBytes / 4), &to, kCacheBytes);
          m++;
          const uint64_t units = (uint64_t)page_size * (uint64_t)c.row_bytes / unit;
          most = units > most ? units : most;
          least = units < least ? units : least;
          total += units * n;
        }
        if (m == 0) break;
        uint32_t* pairs = p.words + m * (kCacheBytes / 4);
        for (int32_t i = 0; i < n; i++) {
          pairs[2 * i] = (uint32_t)src[p0 + i];
          pairs[2 * i + 1] = (uint32_t)dst[p0 + i];
          if (rows) pairs[2 * n + i] = (uint32_t)rows[p0 + i];
        }
        p.table = block_table; p.table_stride = bt_stride; p.table_rows = bt_rows; p.table_cols = bt_cols;
        p.num_caches = m; p.num_pairs = n; p.page_size = page_size; p.part = rows != nullptr;
        const bool past = unit == 16 && total * 16 >= kPast;
        // smaller units: up to sixteen to a thread where every CU has 32 workgroups all the same
        uint64_t piece = unit == 16 && !past ? 512 : 256;
        while (unit < 16 && piece < 4096 && piece * 256 * 32 < total) piece *= 2;
        // Workgroups go to the eight XCDs in turn.  Where pages end at different pieces an odd number of them has a page's first ones, which all of
        // them have, on every XCD: 6 pairs x 27 + 27 caches of 128 and 16 KB, filled rows, 16 / 17 pieces 7.5 / 6.1 us.
        unsigned pieces = (unsigned)((most + piece - 1) / piece);
        if (pieces > 1 && (rows || least != most)) pieces |= 1;
        p.piece = (int32_t)piece;
        const dim3 grid(pieces, (unsigned)m, (unsigned)(n + (table ? 1 : 0)));
        table = false;
        if (past) hipLaunchKernelGGL((pages::copy_pages_kernel<u32x4, true>), grid, dim3(256), 0, stream, p);
        else if (unit == 16) hipLaunchKernelGGL((pages::copy_pages_kernel<u32x4, false>), grid, dim3(256), 0, stream, p);
        else if (unit == 4) hipLaunchKernelGGL((pages::copy_pages_kernel<uint32_t, false>), grid, dim3(256), 0, stream, p);
        else hipLaunchKernelGGL((pages::copy_pages_kernel<uint8_t, false>), grid, dim3(256), 0, stream, p);
        const int rc = check_launch(me);
        if (rc != MLA_OK) return rc;
      }
    }
  }
  return MLA_OK;
}
