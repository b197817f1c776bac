// The rows of an accepted path moved to the places behind the context, in all layers' caches at once, when a step's drafted tokens have been judged.
//
//   row(c + d) = row(c + accepted[d])   for d < kept, every cache of the list and every request b; its new length is c + kept
//   row(x): the cache row of a request's place x by its block table;  kept: how many of the first num_accepted entries are each larger than the one
//   before it, places of the request (c + accepted[d] < seq_lens[b]), and in pages that there are
// A path goes down a tree whose tokens stand behind their parents, so accepted[d] >= d, and a row that is overwritten is no later one's source.
//
// What bounds it: few rows of each request, read and written once, behind two dependent reads (the path, its pages).  A lane takes a granule's column of
// one request in one cache, in all its rows: reads in front of writes without a wait for anyone else.
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
  int32_t batch, lanes_shift;                                // log2 of the lanes that a request's row takes in a wavefront
};

template <typename V>
__global__ __launch_bounds__(256) void keep_rows_kernel(const Params p) {
  constexpr int kAtOnce = 8;
  const int lane = threadIdx.x & ((1 << p.lanes_shift) - 1);
  const int64_t b = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> p.lanes_shift;
  if (b >= p.batch) return;
  const Cache c = p.caches[blockIdx.y];
  const uint32_t at = (blockIdx.z << p.lanes_shift) + lane;  // the lane's granule of a row
  const bool mine = at < c.row_bytes / sizeof(V), tells = p.kept && blockIdx.y == 0 && at == 0;
  if (!mine && !tells) return;
  const int ctx = p.context[b], len = p.lens[b];
  int n = p.num[b];
  n = ctx < 0 || n < 0 ? 0 : n < p.most ? n : p.most;
  int last = -1, kept = 0;
  GLOBAL char* column = (GLOBAL char*)c.base + (int64_t)at * sizeof(V);
  struct Row { bool there; int64_t at; };
  auto row = [&](int64_t place) {
    const int64_t pi = p.page_shift >= 0 ? place >> p.page_shift : place / p.page_size;
    if (place < 0 || pi >= p.cols) return Row{false, 0};
    const int32_t page = p.table[b * p.table_stride + pi];
    return Row{page >= 0 && page < p.num_pages, page * c.page_stride + (place - pi * p.page_size) * (int64_t)c.row_stride};
  };
  for (int d0 = 0; d0 < n; d0 += kAtOnce) {
    int from[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; k++) from[k] = d0 + k < n ? p.accepted[b * p.accepted_stride + d0 + k] : -1;
    Row src[kAtOnce], dst[kAtOnce];
    V v[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; k++) {
      const int64_t place = (int64_t)ctx + from[k];
      src[k] = row(from[k] >= 0 && place < len ? place : -1);
      dst[k] = row((int64_t)ctx + d0 + k);
    }
    bool good = true;
#pragma unroll
    for (int k = 0; k < kAtOnce; k++) {
      good = good && from[k] > last && src[k].there && dst[k].there;
      last = from[k];
      kept += good;
      if (from[k] == d0 + k) src[k].there = false;           // (there already)
      else src[k].there = good;
      if (mine && src[k].there) v[k] = *(const GLOBAL V*)(column + src[k].at);
    }
#pragma unroll
    for (int k = 0; k < kAtOnce; k++)
      if (mine && src[k].there) *(GLOBAL V*)(column + dst[k].at) = v[k];
    if (!good) break;
  }
  if (tells) p.kept[b] = ctx < 0 ? ctx : ctx + kept;
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
      int64_t most = 1;
      for (; next < num_caches && m < keep::kCaches; next++) {
        const mlahip_page_cache& c = caches[next];
        const uint64_t bits = (uint64_t)(uintptr_t)c.base | (uint64_t)c.page_stride_bytes | (uint64_t)c.row_stride_bytes | (uint64_t)c.row_bytes;
        if ((bits & 15 ? bits & 3 ? 1 : 4 : 16) != unit) continue;
        p.caches[m++] = keep::Cache{(char*)c.base, c.page_stride_bytes, (uint32_t)c.row_bytes, (uint32_t)c.row_stride_bytes};
        most = c.row_bytes / unit > most ? c.row_bytes / unit : most;
      }
      if (m == 0) break;
      p.lanes_shift = 0;
      while (p.lanes_shift < 6 && (1 << p.lanes_shift) < most) p.lanes_shift++;
      const int64_t groups = (((int64_t)batch << p.lanes_shift) + 255) / 256, pieces = (most + (1 << p.lanes_shift) - 1) >> p.lanes_shift;
      const dim3 grid((unsigned)groups, (unsigned)m, (unsigned)pieces);
      if (unit == 16) hipLaunchKernelGGL((keep::keep_rows_kernel<u32x4>), grid, dim3(256), 0, stream, p);
      else if (unit == 4) hipLaunchKernelGGL((keep::keep_rows_kernel<uint32_t>), grid, dim3(256), 0, stream, p);
      else hipLaunchKernelGGL((keep::keep_rows_kernel<uint8_t>), grid, dim3(256), 0, stream, p);
      if (int e = check_launch(me)) return e;
      p.kept = nullptr;
    }
  }
  return MLA_OK;
}
