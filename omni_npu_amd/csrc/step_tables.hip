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
//
// A few KB: what takes time is what waits for something else.  A launch of this takes 3.3 us when it does nothing for tokens, of which one is the first
// loads' way; so all of a request's numbers are asked for at once, one scan adds up what is given back and what is needed (the others only where a
// list is too short), what tokens look up lies in LDS, parents too (a tree ten deep is ten loads behind each other), and a token's page is under way
// meanwhile.  us, where no page moves: one token 4.1, 67 requests of 26 tokens as trees 6.2, 500 of up to 64 8.4 (pages 3.3, tokens 5), 16 000 tokens of
// prompts 6.3; loads where they are used: 4.5, 9.0, 9.3, 6.9.  Kernels alone, none / the steps' pages taken: trees of 67 6.0 / 8.4 (104 pages, and 6 back), the
// pages' launch of 500 requests 3.4 / 4.0, of nine prompts 3.2 / 4.2 (128 pages).
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

typedef const __attribute__((address_space(1))) int32_t* Ints;
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

// What a workgroup's tokens look up, in LDS: the beginnings of the requests, every ``apart``th of them where they are many, contexts and lengths of up to
// kFew requests, and the parents of its tokens and of up to kBack in front of them (a tree's, whose bits there are words for).
constexpr int kFew = kThreads, kBack = 512;
template <int kTokens> struct Known {
  int32_t begin[kSamples], ctx[kFew], len[kFew], up[kTokens + kBack];
};
__device__ __forceinline__ int apart_of(const Params& p) { return p.batch / kSamples + 1; }
template <int kTokens> __device__ __forceinline__ void know(const Params& p, Known<kTokens>& known, int64_t first, bool lengths, int threads) {
  if (p.qsl) {
    const int apart = apart_of(p);
    for (int i = threadIdx.x; i * apart <= p.batch; i += threads) known.begin[i] = p.qsl[i * apart];
  }
  if (lengths && p.batch <= kFew) {
    for (int i = threadIdx.x; i < p.batch; i += threads) {
      known.ctx[i] = p.context[i];
      if (p.held) known.len[i] = p.seq_lens[i];
    }
  }
  if (p.parents) {
    const int64_t from = first > kBack ? first - kBack : 0, most = p.num_tokens - from;
    for (int i = threadIdx.x; i < kTokens + kBack && i < most; i += threads) known.up[i] = p.parents[from + i];
  }
}

// Token t, of a workgroup's kTokens from ``first`` on.
template <int kTokens> __device__ __forceinline__ void token(const Params& p, const Known<kTokens>& known, int64_t first, int64_t t) {
  int b = 0;
  int64_t begin = 0, n = 0;
  if (p.batch > 0) {
    if (p.qsl) {                                             // the last request that begins at or in front of t
      const int apart = apart_of(p);
      int lo = 0, hi = (p.batch - 1) / apart;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (known.begin[mid] <= t) lo = mid;
        else hi = mid - 1;
      }
      if (apart == 1) {
        begin = known.begin[lo];
        n = known.begin[lo + 1] - begin;
      } else {
        lo *= apart;
        hi = lo + apart - 1 < p.batch - 1 ? lo + apart - 1 : p.batch - 1;
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (p.qsl[mid] <= t) lo = mid;
          else hi = mid - 1;
        }
        begin = p.qsl[lo];
        n = p.qsl[lo + 1] - begin;
      }
      b = lo;
    } else {
      const uint32_t at = (uint32_t)t / (uint32_t)p.q_len;   // (there are fewer than 2^31 tokens)
      b = at < (uint32_t)p.batch ? (int)at : p.batch - 1;
      begin = (int64_t)b * p.q_len;
      n = p.q_len;
    }
  }
  const int64_t i = t - begin;
  int32_t ctx = -1;
  if (n > 0 && i >= 0 && i < n && begin >= 0) ctx = p.batch <= kFew ? known.ctx[b] : ((Ints)p.context)[b];
  // (its page is under way while the parents are followed)
  int32_t page = -1;
  uint32_t row = 0;
  if (ctx >= 0) {                                            // (idle places and rows behind the last request: none)
    const uint32_t place = (uint32_t)ctx + (uint32_t)i, col = page_of(p, place);
    const int64_t len = ctx + n;
    const bool fits = !p.held || (p.batch <= kFew ? known.len[b] : ((Ints)p.seq_lens)[b]) == (len < 0x7fffffff ? len : 0x7fffffff);
    if (col < (uint32_t)p.cols && fits) page = p.table[b * p.table_stride + col];
    row = place - col * (uint32_t)p.page_size;
  }
  int64_t depth = i;
  if (p.parents) {
    uint64_t* out = p.visible + t * p.visible_stride;
    const int64_t from = first > kBack ? first - kBack : 0;
    uint64_t bits = 0;
    int w = p.words - 1;
    if (ctx >= 0) {
      // up the parents, whose numbers fall
      int32_t at = (int32_t)i;
      if (p.words == 1 && n <= 64 && begin >= from) {
        const int32_t* up = known.up + (begin - from);
        depth = -1;
        int32_t next = at;
        do {
          at = next;
          bits |= 1ull << at;
          depth++;
          next = up[at];
        } while (next >= 0 && next < at);
      } else {                                               // words from the last one on
        const int32_t apart = (int32_t)(begin - from);
        depth = -1;
        while (true) {
          if (at >> 6 < p.words) {
            for (; w > at >> 6; w--) {
              out[w] = bits;
              bits = 0;
            }
            bits |= 1ull << (at & 63);
          }
          depth++;
          const int32_t next = apart + at >= 0 ? known.up[apart + at] : ((Ints)p.parents)[begin + at];
          if (next < 0 || next >= at) break;
          at = next;
        }
      }
    }
    for (; w >= 0; w--) {
      out[w] = bits;
      bits = 0;
    }
  }
  p.positions[t] = ctx >= 0 ? ctx + depth : 0;
  p.slots[t] = page >= 0 ? (int64_t)page * p.page_size + row : -1;
}

// Sums over a workgroup's threads of two values, up to each thread's and whole.
struct Sums { int a, b, all_a, all_b; };
__device__ __forceinline__ Sums scan(int a, int b, int2* parts) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  a = wave_incl_scan_dpp(a);
  b = wave_incl_scan_dpp(b);
  if (lane == 63) parts[wave] = int2{a, b};
  __syncthreads();
  int all_a = 0, all_b = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; w++) {
    const int2 x = parts[w];
    a += w < wave ? x.x : 0;
    b += w < wave ? x.y : 0;
    all_a += x.x;
    all_b += x.y;
  }
  __syncthreads();
  return {a, b, all_a, all_b};
}

// Pages: every request's, by one workgroup, kThreads of them at a time; a thread's own stays in registers where that is all there are.
struct Room { int2 parts[kThreads / 64]; int upto[kThreads], end[kThreads]; };
// A page or a few to a request are its thread's.  More: a page to a thread, which finds the request by its sum.  us, one request that ends with 512 pages by
// its thread / by all 50-59 / 4.5, with 8192 815 / 6.4, 64 with 512 98 / 25, 64 with three 4.4 / 5.0.
constexpr int kOwn = 2, kOwnBack = 4;
__device__ void pages(const Params& p, Room& room, int32_t* ctx, int32_t* len) {
  const int tid = threadIdx.x;
  const int there = *p.num_free;
  struct { Length x; int t, h, give, need; } m;
  Sums s;                                                    // of pages given back and needed
  auto look = [&](int base) {
    m = {{0, 0}, 0, 0, 0, 0};
    if (base + tid < p.batch) {
      m.x = length_of(p, base + tid);
      m.t = pages_of(p, m.x.len);
      m.h = held_of(p, base + tid);
      m.give = m.h > m.t ? m.h - m.t : 0;                    // (t < h: it fits the table)
      m.need = m.t > m.h && m.t <= p.cols ? m.t - m.h : 0;
    }
    s = scan(m.give, m.need, room.parts);
  };
  auto each = [&](auto f) {
    for (int base = 0; base < p.batch; base += kThreads) {
      if (p.batch > kThreads) look(base);
      f(base);
    }
  };
  if (p.batch <= kThreads) look(0);
  int free = there < 0 ? 0 : there < p.capacity ? there : p.capacity;
  // pages that go back: how many in all, then each to its place (all sums of pages are below 2^31, as tables have fewer, with those of the list they need not be)
  const int left = p.capacity - free;
  int back = 0, before = 0;
  // page k of a request's that end at room.upto: f(the request's row, the page's entry in it)
  auto spread = [&](int base, int all, auto fits, auto f) {
    const int rows = p.batch - base < kThreads ? p.batch - base : kThreads;
    for (int k = tid; k < all; k += kThreads) {
      int lo = 0, hi = rows - 1;
      while (lo < hi) {                                      // the first whose sum is above k
        const int mid = (lo + hi) >> 1;
        if (room.upto[mid] > k) hi = mid;
        else lo = mid + 1;
      }
      if (fits(room.upto[lo])) f(k, p.table + (base + lo) * p.table_stride + room.end[lo] - (room.upto[lo] - k));
    }
  };
  each([&](int) { back += s.all_a; });
  if (back > left) {
    back = 0;
    each([&](int) {
      back += scan(before + s.a <= left ? m.give : 0, 0, room.parts).all_a;
      before += s.all_a;
    });
    before = 0;
  }
  if (back > 0) {
    each([&](int base) {
      const bool goes = m.give > 0 && before + s.a <= left;
      if (goes) p.held[base + tid] = m.t;
      if (s.all_a > 0) {
        room.upto[tid] = s.a;
        room.end[tid] = m.h;
        const int top = free + back - 1 - before;
        if (__syncthreads_or(m.give > kOwnBack)) {
          spread(base, s.all_a, [&](int upto) { return before + upto <= left; }, [&](int k, const int32_t* at) { p.free_pages[top - k] = *at; });
          __syncthreads();
        } else if (goes) {
          const int32_t* row = p.table + (base + tid) * p.table_stride + m.t;
          int32_t mine[kOwnBack];
#pragma unroll
          for (int k = 0; k < kOwnBack; k++) mine[k] = row[k < m.give ? k : 0];
#pragma unroll
          for (int k = 0; k < kOwnBack; k++)
            if (k < m.give) p.free_pages[top - (s.a - m.give) - k] = mine[k];
        }
      }
      before += s.all_a;
    });
    free += back;
    __syncthreads();
  }
  // pages that are taken
  int taken = 0;
  before = 0;
  each([&](int base) {
    const bool got = m.need == 0 || before + s.b <= free;
    if (base + tid < p.batch) {
      const int32_t now = m.t <= p.cols && got ? m.x.len : m.x.ctx;
      p.seq_lens[base + tid] = now;
      if (p.batch <= kFew) {
        ctx[tid] = m.x.ctx;
        len[tid] = now;
      }
      if (m.need > 0 && got) p.held[base + tid] = m.t;
    }
    if (s.all_b > 0) {
      room.upto[tid] = s.b;
      room.end[tid] = m.t;
      const int all = s.all_b;
      if (__syncthreads_or(m.need > kOwn)) {
        spread(base, all, [&](int upto) { return before + upto <= free; }, [&](int k, int32_t* at) { *at = p.free_pages[free - 1 - before - k]; });
      } else if (got) {
#pragma unroll
        for (int k = 0; k < kOwn; k++)
          if (k < m.need) p.table[(base + tid) * p.table_stride + m.h + k] = p.free_pages[free - 1 - before - (s.b - m.need) - k];
      }
      taken += before + all <= free ? all : scan(got ? m.need : 0, 0, room.parts).all_a;
      before += all;
      __syncthreads();
    }
  });
  if (tid == 0) *p.num_free = free - taken;
}

// Tokens that the workgroup of the pages does as well.  us, together / in a launch of their own: 1500 tokens in trees 6.0 / 6.8, 2000 6.7 / 7.0, 3000
// 7.9 / 7.0; 2000 tokens of four requests 5.0 / 7.0, 4000 6.1 / 7.0; of as many requests 3000 11.2 / 10.3.
constexpr int kTogether = 2048, kBlock = 256;

__global__ __launch_bounds__(kThreads) void step_pages_kernel(const Params p, int with_tokens) {
  __shared__ Room room;
  __shared__ Known<kTogether> known;
  if (with_tokens) know(p, known, 0, false, kThreads);
  pages(p, room, known.ctx, known.len);
  if (!with_tokens) return;
  __syncthreads();
  for (int64_t t = threadIdx.x; t < p.num_tokens; t += kThreads) token(p, known, 0, t);
}

__global__ __launch_bounds__(kBlock) void step_tokens_kernel(const Params p) {
  __shared__ Known<kBlock> known;
  const int64_t first = (int64_t)blockIdx.x * kBlock, t = first + threadIdx.x;
  know(p, known, first, true, kBlock);
  __syncthreads();
  if (!p.held && t < p.batch) p.seq_lens[t] = length_of(p, (int)t).len;
  if (t < p.num_tokens) token(p, known, first, t);
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
  const bool together = num_tokens <= tables::kTogether;
  if (pages) {
    hipLaunchKernelGGL(tables::step_pages_kernel, dim3(1), dim3(tables::kThreads), 0, stream, p, (int)together);
    if (int e = check_launch(me)) return e;
    if (together) return MLA_OK;
  }
  const int64_t n = num_tokens > batch ? num_tokens : batch;
  hipLaunchKernelGGL(tables::step_tokens_kernel, dim3((unsigned)((n + tables::kBlock - 1) / tables::kBlock)), dim3(tables::kBlock), 0, stream, p);
  return check_launch(me);
}
