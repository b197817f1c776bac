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
#include <algorithm>
#include <new>

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

// ---- caches that share memory (on the host): two moves of the same bytes would take each other's results for what they read ----
// A cache as blocks that lie ``outer`` apart, each of rows ``inner`` apart: pages of rows, or, where these lie inside rows, rows of pages.
struct Layout {
  int64_t begin, end;                                        // of all of it
  int64_t outer, inner, row;
  int32_t blocks, rows;
  int64_t block() const { return (rows - 1) * inner + row; }
};
bool layout_of(const mlahip_page_cache& c, int32_t pages, int32_t page_size, Layout* x) {
  const int64_t begin = (int64_t)(uintptr_t)c.base;
  if (pages == 1) *x = {begin, 0, c.row_stride_bytes, 0, c.row_bytes, page_size, 1};
  else if (page_size == 1) *x = {begin, 0, c.page_stride_bytes, 0, c.row_bytes, pages, 1};
  else if (c.page_stride_bytes >= c.row_stride_bytes) *x = {begin, 0, c.page_stride_bytes, c.row_stride_bytes, c.row_bytes, pages, page_size};
  else *x = {begin, 0, c.row_stride_bytes, c.page_stride_bytes, c.row_bytes, page_size, pages};
  int64_t size;
  return !__builtin_mul_overflow((int64_t)(x->blocks - 1), x->outer, &size) && !__builtin_add_overflow(size, x->block(), &size) &&
         !__builtin_add_overflow(begin, size, &x->end);
}
int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0); }
// A block of a and one of b, which begins ``apart`` behind it.
bool blocks_meet(const Layout& a, const Layout& b, int64_t apart) {
  if (apart >= a.block() || apart + b.block() <= 0) return false;
  const auto last_in_front_of = [&](int64_t end, int32_t rows) {   // b's last row that begins in front of ``end``, of so many
    if (rows == 1) return (int64_t)(apart < end ? 0 : -1);
    const int64_t r = floor_div(end - 1 - apart, b.inner);
    return r < rows - 1 ? r : (int64_t)rows - 1;
  };
  if (a.inner == b.inner && a.rows == b.rows) {              // by how many rows b's lie further: -rows < k < rows
    if (a.rows == 1) return true;                            // (two rows that overlap, as said above)
    const int64_t k = floor_div(a.row - 1 - apart, a.inner), most = k < a.rows - 1 ? k : a.rows - 1;
    return most > -(int64_t)a.rows && apart + most * a.inner + b.row > 0;
  }
  for (int64_t i = 0; i < a.rows; i++) {
    const int64_t at = i * a.inner, r = last_in_front_of(at + a.row, b.rows);
    if (r >= 0 && apart + r * b.inner + b.row > at) return true;
  }
  return false;
}
// Blocks that lie differently far apart are not looked through: they are taken to share memory where one cache begins in the other.
bool caches_meet(const Layout& a, const Layout& b) {
  if (a.end <= b.begin || b.end <= a.begin) return false;
  if (a.outer != b.outer || a.blocks != b.blocks) return true;
  if (a.blocks == 1) return blocks_meet(a, b, b.begin - a.begin);
  const int64_t n = floor_div(b.begin - a.begin, a.outer), apart = b.begin - a.begin - n * a.outer;
  const auto some = [&](int64_t by) { return by > -(int64_t)a.blocks && by < a.blocks; };
  return (some(n) && blocks_meet(a, b, apart)) || (some(n + 1) && blocks_meet(a, b, apart - a.outer));
}
// Two of them that share memory; false: none do.  In order of their beginnings, and those that lie in one another (of one storage) as pieces of a block, or of a
// row, where they are such pieces, so that each is held against the next one alone: 128 caches of one storage take 2 us; each against
// each, as where rows of two strides lie between each other, 64 take 66.
struct Place { int64_t at; int32_t of; };
void in_order(Place* x, int32_t n) {
  const auto less = [](const Place& a, const Place& b) { return a.at < b.at; };
  if (!std::is_sorted(x, x + n, less)) std::sort(x, x + n, less);
}
bool any_meet(const Layout* all, Place* places, int32_t n, int32_t* one, int32_t* other) {
  for (int32_t i = 0; i < n; i++) places[i] = {all[i].begin, i};
  in_order(places, n);
  for (int32_t i = 0, next; i < n; i = next) {
    const Layout& first = all[places[i].of];
    int64_t end = first.end;
    bool alike = true, rows = true;
    for (next = i + 1; next < n && places[next].at < end; next++) {
      const Layout& x = all[places[next].of];
      end = x.end > end ? x.end : end;
      alike = alike && x.outer == first.outer;
      rows = rows && x.inner == first.inner && x.rows == first.rows;
    }
    const int32_t m = next - i;
    Place* x = places + i;
    if (m == 1) continue;
    // places modulo a stride, each with what it takes there: apart from the next one, and the last from the first
    const auto apart = [&](int64_t stride, auto size) {
      for (int32_t k = 0; k < m; k++) x[k].at = (all[x[k].of].begin - first.begin) % stride;
      in_order(x, m);
      for (int32_t k = 0; k < m; k++)
        if (x[k].at + size(all[x[k].of]) > (k + 1 < m ? x[k + 1].at : x[0].at + stride)) return false;
      return true;
    };
    if (alike && apart(first.outer, [](const Layout& y) { return y.block(); })) continue;
    if (alike && rows && first.rows > 1 && first.outer % first.inner == 0 && apart(first.inner, [](const Layout& y) { return y.row; })) continue;
    for (int32_t k = 0; k < m; k++)
      for (int32_t l = k + 1; l < m; l++)
        if (caches_meet(all[x[k].of], all[x[l].of])) {
          *one = x[k].of < x[l].of ? x[k].of : x[l].of;
          *other = x[k].of < x[l].of ? x[l].of : x[k].of;
          return true;
        }
  }
  return false;
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
  {
    constexpr int32_t kFew = 256;
    keep::Layout few[kFew], *layouts = few;
    keep::Place few_places[kFew], *places = few_places;
    if (num_caches > kFew) {
      layouts = new (std::nothrow) keep::Layout[num_caches];
      places = new (std::nothrow) keep::Place[num_caches];
    }
    int32_t one = 0, other = 0, past = -1;
    bool meet = false;
    const bool room = layouts && places;
    if (room) {
      for (int32_t i = 0; i < num_caches && past < 0; i++)
        if (!keep::layout_of(caches[i], (int32_t)num_pages, page_size, layouts + i)) past = i;
      meet = past < 0 && keep::any_meet(layouts, places, num_caches, &one, &other);
    }
    if (num_caches > kFew) {
      delete[] layouts;
      delete[] places;
    }
    MLA_REQUIRE(room, MLA_ERR_UNSUPPORTED, "%s: no memory to look through %d caches", me, num_caches);
    MLA_REQUIRE(past < 0, MLA_ERR_SHAPE, "%s: cache %d: pages %lld apart end past all addresses", me, past, (long long)caches[past < 0 ? 0 : past].page_stride_bytes);
    MLA_REQUIRE(!meet, MLA_ERR_UNSUPPORTED, "%s: caches %d and %d share memory", me, one, other);
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
