// What a step reads besides its queries, from the requests' lengths: pages into the block tables and back out of them, lengths, positions, slots, and
// for tokens drafted as trees which tokens each one sees.
//
//   request b: c cached tokens (below 0: an idle place, no tokens), n new ones, L = c + n, pages h, t = ceil(L / page)
//   h > t      pages t .. h of its table go back to the list of free ones, in the order in which they would be taken from it again
//   h < t      pages from the list's end, in the order of the requests; from the first request that there are too few for on, none gets any
//   token i    slot = table[(c + i) / page] * page + (c + i) % page, position = c + its depth (without parents: i)
//   sees       itself and the tokens that its parents lead to, a bit each
//
// A list's order hangs on all requests in front of one: sums over the requests, by one workgroup, which changes the list, the tables and the counts.  The
// tokens of larger steps follow in a launch of their own, when these stand.
#include "mla_common.hpp"
#include "../../include/mla_hip.h"

namespace mlahip {
namespace tables {

struct Params {
  const int32_t *context, *qsl;
  int32_t q_len, batch;
  int32_t* table; int64_t table_stride; int32_t cols, page_size, page_shift;   // log2 of the page, -1 where it is no power of two
  int32_t* seq_lens;
  int64_t *positions, *slots; int64_t num_tokens;
  const int32_t* parents;                                    // or null
  uint64_t* visible; int64_t visible_stride; int32_t words;
  int32_t *held, *free_pages, *num_free; int32_t capacity;   // or null
};

constexpr int kThreads = 1024, kSamples = 4096;

// Tokens of request b, however its entries lie: at least none.
__device__ __forceinline__ int64_t tokens_of(const Params& p, int b) {
  if (!p.qsl) return p.q_len;
  const int64_t n = (int64_t)p.qsl[b + 1] - p.qsl[b];
  return n > 0 ? n : 0;
}
struct Length { int32_t ctx, len; };                         // (an idle place: -1, 0)
__device__ __forceinline__ Length length_of(const Params& p, int b) {
  const int32_t c = p.context[b];
  if (c < 0) return {c, 0};
  const int64_t len = c + tokens_of(p, b);
  return {c, len < 0x7fffffff ? (int32_t)len : 0x7fffffff};
}
__device__ __forceinline__ uint32_t page_of(const Params& p, uint32_t place) {
  return p.page_shift >= 0 ? place >> p.page_shift : place / (uint32_t)p.page_size;
}
__device__ __forceinline__ int pages_of(const Params& p, int32_t len) { return len > 0 ? (int)page_of(p, (uint32_t)len - 1) + 1 : 0; }
__device__ __forceinline__ int held_of(const Params& p, int b) {
  const int h = p.held[b];
  return h < 0 ? 0 : h < p.cols ? h : p.cols;
}

// The tokens t of a workgroup's threads; samples: every ``apart``th entry of qsl.
__device__ __forceinline__ void token(const Params& p, int64_t t, const int32_t* samples, int apart) {
  int b = 0;
  int64_t begin = 0, n = 0;
  if (p.batch > 0) {
    if (p.qsl) {                                             // the last request that begins at or in front of t
      int lo = 0, hi = (p.batch - 1) / apart;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (samples[mid] <= t) lo = mid;
        else hi = mid - 1;
      }
      lo *= apart;
      hi = lo + apart - 1 < p.batch - 1 ? lo + apart - 1 : p.batch - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (p.qsl[mid] <= t) lo = mid;
        else hi = mid - 1;
      }
      b = lo;
      begin = p.qsl[b];
      n = tokens_of(p, b);
    } else {
      const int64_t at = t / p.q_len;
      b = at < p.batch ? (int)at : p.batch - 1;
      begin = (int64_t)b * p.q_len;
      n = p.q_len;
    }
  }
  const int64_t i = t - begin;
  int64_t position = 0, slot = -1;
  const bool there = n > 0 && i >= 0 && i < n && begin >= 0 && p.context[b] >= 0;
  int64_t depth = i;
  if (p.parents) {
    uint64_t* row = p.visible + t * p.visible_stride;
    if (there) {
      // up the parents, whose numbers fall: words from the last one on
      const int32_t* up = p.parents + begin;
      int64_t at = i;
      uint64_t bits = 0;
      int w = p.words - 1;
      depth = -1;
      while (true) {
        if (at >> 6 < p.words) {
          for (; w > (int)(at >> 6); w--) {
            row[w] = bits;
            bits = 0;
          }
          bits |= 1ull << (at & 63);
        }
        depth++;
        const int64_t next = up[at];
        if (next < 0 || next >= at) break;
        at = next;
      }
      for (; w >= 0; w--) {
        row[w] = bits;
        bits = 0;
      }
    } else {
      for (int w = 0; w < p.words; w++) row[w] = 0;
    }
  }
  if (there) {
    const Length x = length_of(p, b);
    position = x.ctx + depth;
    const uint32_t place = (uint32_t)x.ctx + (uint32_t)i, col = page_of(p, place);
    if (col < (uint32_t)p.cols && (!p.held || p.seq_lens[b] == x.len)) {
      const int32_t page = p.table[b * p.table_stride + col];
      if (page >= 0) slot = (int64_t)page * p.page_size + (place - col * (uint32_t)p.page_size);
    }
  }
  p.positions[t] = position;
  p.slots[t] = slot;
}

__device__ __forceinline__ int apart_of(const Params& p) { return p.batch > kSamples ? (p.batch + kSamples - 1) / kSamples : 1; }
__device__ __forceinline__ void take_samples(const Params& p, int32_t* samples, int threads) {
  if (!p.qsl) return;
  const int apart = apart_of(p);
  for (int i = threadIdx.x; i * apart < p.batch; i += threads) samples[i] = p.qsl[i * apart];
}

// Inclusive sums over a workgroup's threads, and the whole one.
struct Sum { int upto, all; };
__device__ __forceinline__ Sum scan(int v, int* parts) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int mine = wave_incl_scan_dpp(v);
  if (lane == 63) parts[wave] = mine;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; w++) {
    before += w < wave ? parts[w] : 0;
    all += parts[w];
  }
  __syncthreads();
  return {before + mine, all};
}

// Pages: every request's, by one workgroup.
__device__ void pages(const Params& p, int* parts, int* upto) {
  const int tid = threadIdx.x;
  const int there = *p.num_free;
  int free = there < 0 ? 0 : there < p.capacity ? there : p.capacity;
  // pages that go back: how many in all, then each to its place
  int back = 0;
  auto gives = [&](int b) {
    if (b >= p.batch) return 0;
    const int t = pages_of(p, length_of(p, b).len), h = held_of(p, b);
    return h > t ? h - t : 0;                                // (t < h: it fits the table)
  };
  int before = 0;
  for (int base = 0; base < p.batch; base += kThreads) {
    const int n = gives(base + tid);
    const Sum s = scan(n, parts);
    back += scan(before + s.upto + free <= p.capacity ? n : 0, parts).all;
    before += s.all;
  }
  if (before > 0) {
    before = 0;
    for (int base = 0; base < p.batch; base += kThreads) {
      const int b = base + tid, n = gives(b);
      const Sum s = scan(n, parts);
      if (n > 0 && before + s.upto + free <= p.capacity) {
        const int t = held_of(p, b) - n, first = free + back - 1 - (before + s.upto - n);
        for (int k = 0; k < n; k++) p.free_pages[first - k] = p.table[b * p.table_stride + t + k];
        p.held[b] = t;
      }
      before += s.all;
    }
    free += back;
    __syncthreads();
  }
  // pages that are taken
  int taken = 0;
  before = 0;
  for (int base = 0; base < p.batch; base += kThreads) {
    const int b = base + tid;
    int need = 0, t = 0, h = 0;
    Length x{0, 0};
    if (b < p.batch) {
      x = length_of(p, b);
      t = pages_of(p, x.len);
      h = held_of(p, b);
      need = t > h && t <= p.cols ? t - h : 0;
    }
    const Sum s = scan(need, parts);
    const bool got = need == 0 || before + s.upto <= free;
    if (b < p.batch) {
      p.seq_lens[b] = t <= p.cols && got ? x.len : x.ctx;
      if (need > 0 && got) p.held[b] = t;
    }
    taken += scan(need > 0 && got ? need : 0, parts).all;
    if (s.all > 0) {
      // a page to a thread: the request that it is for by its sum
      upto[tid] = s.upto;
      __syncthreads();
      const int rows = p.batch - base < kThreads ? p.batch - base : kThreads;
      for (int k = tid; k < s.all; k += kThreads) {
        int lo = 0, hi = rows - 1;
        while (lo < hi) {                                    // the first whose sum is above k
          const int mid = (lo + hi) >> 1;
          if (upto[mid] > k) hi = mid;
          else lo = mid + 1;
        }
        if (before + upto[lo] > free) continue;
        const int first = lo > 0 ? upto[lo - 1] : 0, n = upto[lo] - first;
        const Length y = length_of(p, base + lo);
        p.table[(base + lo) * p.table_stride + pages_of(p, y.len) - n + (k - first)] = p.free_pages[free - 1 - before - k];
      }
      __syncthreads();
    }
    before += s.all;
  }
  if (tid == 0) *p.num_free = free - taken;
}

__global__ __launch_bounds__(kThreads) void step_pages_kernel(const Params p, int with_tokens) {
  __shared__ int parts[kThreads / 64], upto[kThreads];
  __shared__ int32_t samples[kSamples];
  if (with_tokens) take_samples(p, samples, kThreads);
  pages(p, parts, upto);
  if (!with_tokens) return;
  __syncthreads();
  for (int64_t t = threadIdx.x; t < p.num_tokens; t += kThreads) token(p, t, samples, apart_of(p));
}

__global__ __launch_bounds__(256) void step_tokens_kernel(const Params p) {
  __shared__ int32_t samples[kSamples];
  take_samples(p, samples, 256);
  __syncthreads();
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (!p.held && t < p.batch) p.seq_lens[t] = length_of(p, (int)t).len;
  if (t < p.num_tokens) token(p, t, samples, apart_of(p));
}

struct Range { const char *begin, *end; };
Range range(const void* at, int64_t bytes) { return {(const char*)at, (const char*)at + (at ? bytes : 0)}; }
bool meet(Range a, Range b) { return a.begin < b.end && b.begin < a.end; }

}  // namespace tables
}  // namespace mlahip
using namespace mlahip;

extern "C" int mlahip_step_tables(const int32_t* context_lens, const int32_t* query_start_loc, int32_t batch, int32_t q_len, int32_t* block_table,
                                  int64_t bt_stride, int32_t max_blocks, int32_t page_size, int32_t* seq_lens, int64_t* positions,
                                  int64_t* slot_mapping, int64_t num_tokens, const int32_t* parents, uint64_t* visible, int64_t visible_stride,
                                  int32_t words, int32_t* num_blocks, int32_t* free_pages, int32_t* num_free, int32_t capacity, hipStream_t stream) {
  const char* me = "mlahip_step_tables";
  MLA_REQUIRE(batch >= 0 && batch < (1 << 24) && q_len >= 1 && page_size >= 1 && max_blocks >= 1 && (batch <= 1 || bt_stride >= max_blocks) &&
                  (int64_t)batch * max_blocks < (1ll << 31) && num_tokens >= 0 && num_tokens < (1ll << 31),
              MLA_ERR_SHAPE, "%s: %d requests of %d tokens, %lld places, tables of %d pages of %d, %lld apart", me, batch, q_len, (long long)num_tokens,
              max_blocks, page_size, (long long)bt_stride);
  MLA_REQUIRE(batch == 0 || (context_lens && block_table && seq_lens), MLA_ERR_NULL, "%s: null pointer argument", me);
  MLA_REQUIRE(num_tokens == 0 || (positions && slot_mapping), MLA_ERR_NULL, "%s: null pointer argument", me);
  MLA_REQUIRE((parents != nullptr) == (visible != nullptr) || num_tokens == 0, MLA_ERR_NULL, "%s: parents and visible go together", me);
  MLA_REQUIRE(batch == 0 || ((num_blocks != nullptr) == (num_free != nullptr) && (free_pages || capacity == 0) && (num_blocks || !free_pages)), MLA_ERR_NULL,
              "%s: num_blocks, free_pages and num_free go together", me);
  MLA_REQUIRE(query_start_loc || num_tokens >= (int64_t)batch * q_len, MLA_ERR_SHAPE, "%s: %lld places for %d requests of %d tokens", me,
              (long long)num_tokens, batch, q_len);
  MLA_REQUIRE(!parents || (words >= 1 && (num_tokens <= 1 || visible_stride >= words) && (query_start_loc || (int64_t)words * 64 >= q_len)),
              MLA_ERR_SHAPE, "%s: %d words for the bits of %d tokens, rows %lld apart", me, words, q_len, (long long)visible_stride);
  MLA_REQUIRE(!num_blocks || capacity >= 0, MLA_ERR_SHAPE, "%s: a list of %d pages", me, capacity);
  // what is written while other threads read the rest
  const int64_t rows = batch > 0 ? batch - 1 : 0;
  const bool pages = batch > 0 && num_blocks != nullptr;
  const tables::Range all[] = {tables::range(seq_lens, batch * 4ll), tables::range(positions, num_tokens * 8), tables::range(slot_mapping, num_tokens * 8),
                               tables::range(parents ? visible : nullptr, num_tokens > 0 ? ((num_tokens - 1) * visible_stride + words) * 8 : 0),
                               tables::range(num_blocks, batch * 4ll), tables::range(free_pages, capacity * 4ll), tables::range(num_free, 4),
                               tables::range(batch > 0 ? block_table : nullptr, (rows * bt_stride + max_blocks) * 4),
                               tables::range(context_lens, batch * 4ll), tables::range(query_start_loc, batch * 4ll + 4),
                               tables::range(parents, num_tokens * 4)};
  for (int i = 0; i < (pages ? 8 : 4); i++)
    for (int k = i + 1; k < 11; k++)
      MLA_REQUIRE(!tables::meet(all[i], all[k]), MLA_ERR_UNSUPPORTED, "%s: a result shares memory with another tensor of the call", me);
  const uintptr_t fours = (uintptr_t)context_lens | (uintptr_t)query_start_loc | (uintptr_t)block_table | (uintptr_t)seq_lens | (uintptr_t)parents |
                          (uintptr_t)num_blocks | (uintptr_t)free_pages | (uintptr_t)num_free;
  MLA_REQUIRE(!(fours & 3) && !(((uintptr_t)positions | (uintptr_t)slot_mapping | (uintptr_t)visible) & 7), MLA_ERR_SHAPE,
              "%s: unaligned pointers", me);
  if (batch == 0 && num_tokens == 0) return MLA_OK;
  tables::Params p{};
  p.context = context_lens; p.qsl = query_start_loc; p.q_len = q_len; p.batch = batch;
  p.table = block_table; p.table_stride = bt_stride; p.cols = max_blocks; p.page_size = page_size;
  p.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz(page_size) : -1;
  p.seq_lens = seq_lens; p.positions = positions; p.slots = slot_mapping; p.num_tokens = num_tokens;
  p.parents = num_tokens > 0 ? parents : nullptr; p.visible = visible; p.visible_stride = visible_stride; p.words = words;
  p.held = pages ? num_blocks : nullptr; p.free_pages = free_pages; p.num_free = num_free; p.capacity = capacity;
  const bool together = num_tokens <= 2048;
  if (pages) {
    hipLaunchKernelGGL(tables::step_pages_kernel, dim3(1), dim3(tables::kThreads), 0, stream, p, (int)together);
    if (int e = check_launch(me)) return e;
    if (together) return MLA_OK;
  }
  const int64_t n = num_tokens > batch ? num_tokens : batch;
  hipLaunchKernelGGL(tables::step_tokens_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, p);
  return check_launch(me);
}
