// A cache in pages: pages dealt to sequences and taken back, keys and values written to them, attention of new tokens over them.
// Declarations: include/marian_hip_ops.h
#include "../../include/marian_hip_ops.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "abi_common.h"
#include "cache_args.h"
#include "cache_attention_kernel.h"
#include "pages_attention.h"

using namespace marian_hip;

namespace {

// ---------------------------------------------------------------- pages dealt and taken back
struct TablesArgs {
  int *table, *held, *free, *free_count;
  const int *lens, *counts;
  int S, row, pages, n, page;
  CacheDivisor by_page, by_n;
  int* slots;
};

// The pages that sequence s lacks for its new tokens, or (TRIM) that lie behind its positions; first: the first one's place in its row.
template <bool TRIM>
__device__ __forceinline__ int pages_moved(const TablesArgs& a, int s, int& first) {
  const int held = clamp_int(a.held[s], 0, a.row);
  const unsigned len = (unsigned)max(a.lens[s], 0);
  if constexpr(TRIM) {
    first = min(held, (int)a.by_page.of(len + a.page - 1));
    return held - first;
  } else {
    const unsigned count = a.counts ? clamp_int(a.counts[s], 0, a.n) : a.n;
    const int need = (int)a.by_page.of(len + count + a.page - 1);   // (less than 2^32: n is at most 2^20)
    first = held;
    return need > a.row ? 0 : max(0, need - held);
  }
}

constexpr int kDealers = 1024;   // threads of a workgroup that deals, a sequence each at a time

// What a workgroup knows of the sequences it deals for.
struct Dealt {
  int before[kDealers + 1];   // where their pages lie in one line of all of them
  int first[kDealers], len[kDealers], count[kDealers];
  int waves[kDealers / 64];
  int most;
};

// The sum of x over the threads before this one; all: over all of them.  In the end `waves` has been read.
__device__ __forceinline__ int dealers_sum_before(Dealt& sh, int x, int& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int sum = (int)lanes_sum((unsigned)x);
  if(lane == 63) sh.waves[wave] = sum;
  __syncthreads();
  int ahead = 0;
  all = 0;
#pragma unroll
  for(int i = 0; i < kDealers / 64; ++i) {
    if(i == wave) ahead = all;
    all += sh.waves[i];
  }
  __syncthreads();
  return ahead + sum - x;
}

// Deals pages and maps slots, or takes pages back (MOVE), and settles the counts (SETTLE).  Where there is little one workgroup does all of it; else
// many move, each finding the sequences' places in the line by itself, and a second launch of one workgroup settles, for until all have
// read the counts none may write them.  A slot's page comes from the stack where the table does not have it yet, so nothing waits for
// the table.  Small calls are a launch and a chain of steps (lengths, sum, page, store): 6 sequences 2.8 us, 2.1 to take back.  513 prompts of up to 2047
// tokens 7.2 us and 4.4 to settle, 3.9 and 2.1 to take back, 256 workgroups (128: 9.1, 512: 8.8); their 4 MB of slots are 1 us of it.
template <bool TRIM, bool MOVE, bool SETTLE>
__global__ __launch_bounds__(kDealers) void pages_deal_kernel(TablesArgs a) {
  __shared__ Dealt sh;
  const int tid = threadIdx.x, available = clamp_int(*a.free_count, 0, a.pages);
  int all = 0, carry = 0, dealt = 0, first;
  if(TRIM && a.S > kDealers) {   // (the last page of the line goes to the bottom)
    int mine = 0;
    for(int s = tid; s < a.S; s += kDealers) mine += pages_moved<TRIM>(a, s, first);
    dealers_sum_before(sh, mine, all);
  }
  for(int base = 0; base < a.S; base += kDealers) {
    const int s = base + tid, here = min(kDealers, a.S - base);
    const int more = tid < here ? pages_moved<TRIM>(a, s, first) : 0;
    int sum;
    const int mine = carry + dealers_sum_before(sh, more, sum);
    if(tid < here) {
      sh.before[tid] = mine;
      sh.first[tid] = first;
      if(!TRIM) {
        sh.len[tid] = max(a.lens[s], 0);
        sh.count[tid] = a.counts ? a.counts[s] : a.n;
      }
    }
    if(tid == 0) sh.before[here] = carry + sum;
    if(TRIM && a.S <= kDealers) all = sum;
    if(!TRIM && mine + more <= available && more > 0) dealt = mine + more;
    __syncthreads();
    if constexpr(MOVE) {
      // A thread to a sequence where each has few pages, or a wave.
      auto move = [&](int q, int j) __attribute__((always_inline)) {
        int* const entry = a.table + (long long)(base + q) * a.row + sh.first[q] + j;
        const int t = sh.before[q] + j;
        if constexpr(TRIM) {
          const long long to = (long long)available + all - 1 - t;
          if(to < a.pages) a.free[to] = *entry;
          *entry = -1;
        } else {
          *entry = a.free[available - 1 - t];
        }
      };
      const int each = TRIM ? 64 : a.n / a.page > 8 ? 64 : 1;
      for(int q = (blockIdx.x * kDealers + tid) / each; q < here; q += gridDim.x * kDealers / each) {
        const int pages = sh.before[q + 1] - sh.before[q];
        if(!TRIM && sh.before[q + 1] > available) continue;
        for(int j = tid % each; j < pages; j += each) move(q, j);
      }
      if constexpr(!TRIM) {
        const unsigned ids = (unsigned)here * a.n;
        for(unsigned id = blockIdx.x * kDealers + tid; id < ids; id += gridDim.x * kDealers) {
          unsigned i, within;
          const int q = (int)a.by_n.of(id, i), j = (int)a.by_page.of((unsigned)sh.len[q] + i, within), k = j - sh.first[q];
          int page = -1;
          if((int)i < sh.count[q] && j < a.row) {
            const bool fresh = k >= 0 && sh.before[q + 1] <= available && k < sh.before[q + 1] - sh.before[q];
            const int* const from = fresh ? a.free + (available - 1 - sh.before[q] - k) : a.table + (long long)(base + q) * a.row + j;
            page = *from;
          }
          a.slots[(long long)base * a.n + id] = (unsigned)page < (unsigned)a.pages ? page * a.page + (int)within : -1;
        }
      }
    }
    carry += sum;
    if constexpr(SETTLE) {
      if(tid < here) {
        if(TRIM) a.held[s] = first;
        else if(more > 0 && mine + more <= available) a.held[s] = first + more;
      }
    }
    __syncthreads();   // (the places in LDS are read)
  }
  if constexpr(SETTLE) {
    if(tid == 0) sh.most = 0;
    __syncthreads();
    if(!TRIM && dealt > 0) atomicMax(&sh.most, dealt);
    __syncthreads();
    if(tid == 0) *a.free_count = TRIM ? (int)min((long long)available + all, (long long)a.pages) : available - sh.most;
  }
}

// ---------------------------------------------------------------- writing
struct WriteArgs {
  unsigned char *k, *v;
  Strides kx, vx;
  const int* slots;
  int heads, page, row_bytes, width;
  unsigned pieces;   // of all rows
  int slots_end;     // of all pages
  CacheDivisor by_units, by_heads, by_n, by_page;
};

// A thread takes a piece of sixteen bytes of a row of keys and of values, kWriteTurns times, all asked for before the first is stored.  A copy:
// memory bounds it.  3 prompts of 2731 tokens, 8 heads of 128 values, bfloat16: 10.8 us, 6.2 TB/s (a large copy: 5.1; these 67 MB stay in the last
// cache); 128 single tokens of 16 heads of 64 values, float32: 2.6 us, a launch and three steps.
constexpr int kWriteTurns = 2;
__global__ __launch_bounds__(256) void pages_write_kernel(const unsigned char* __restrict__ k, const unsigned char* __restrict__ v, WriteArgs a) {
  cache_u4 x[kWriteTurns][2];
  long long to[kWriteTurns];
#pragma unroll
  for(int t = 0; t < kWriteTurns; ++t) {
    const unsigned id = (blockIdx.x * kWriteTurns + t) * 256u + threadIdx.x, mine = min(id, a.pieces - 1);
    unsigned unit, h, i, within;
    const unsigned token = a.by_heads.of(a.by_units.of(mine, unit), h), s = a.by_n.of(token, i);
    const int slot = a.slots[token];
    x[t][0] = *reinterpret_cast<const cache_u4*>(k + (s * a.kx.s + h * a.kx.h + i * a.kx.n) * a.width + 16 * unit);
    x[t][1] = *reinterpret_cast<const cache_u4*>(v + (s * a.vx.s + h * a.vx.h + i * a.vx.n) * a.width + 16 * unit);
    const unsigned page = a.by_page.of((unsigned)max(slot, 0), within);
    to[t] = id < a.pieces && slot >= 0 && slot < a.slots_end
                ? (((long long)page * a.heads + h) * a.page + within) * a.row_bytes + 16 * unit : -1;
  }
#pragma unroll
  for(int t = 0; t < kWriteTurns; ++t) {
    if(to[t] < 0) continue;
    *reinterpret_cast<cache_u4*>(a.k + to[t]) = x[t][0];
    *reinterpret_cast<cache_u4*>(a.v + to[t]) = x[t][1];
  }
}

// ---------------------------------------------------------------- arguments
constexpr int64_t kMaxPage = 4096, kMaxPositions = (1 << 30) - 1;

int check_page(int64_t page) { return page >= 8 && page % 8 == 0 && page <= kMaxPage ? MARIAN_HIP_OK : MARIAN_HIP_ERR_SHAPE; }

int check_pages(const marian_hip_pages* c) {
  if(!c) return MARIAN_HIP_ERR_NULL;
  MH_CHECK(check_type(c->type));
  MH_CHECK(check_page(c->page));
  if(c->pages < 1 || c->heads < 1 || !row_size(c->dk)) return MARIAN_HIP_ERR_SHAPE;
  return c->heads > kMaxHeads || c->pages > kMaxPositions / c->page ? MARIAN_HIP_ERR_RANGE : MARIAN_HIP_OK;
}
int check_pages_memory(const marian_hip_pages* c) {
  if(!c->k || !c->v) return MARIAN_HIP_ERR_NULL;
  return aligned(c->k, 16) && aligned(c->v, 16) ? MARIAN_HIP_OK : MARIAN_HIP_ERR_ALIGN;
}
int64_t pages_bytes(const marian_hip_pages* c) { return c->pages * c->heads * c->page * c->dk * width_of(c->type); }

int check_tables(const marian_hip_page_tables* t, int64_t page) {
  if(!t) return MARIAN_HIP_ERR_NULL;
  MH_CHECK(check_page(page));
  if(t->sequences < 0 || t->row < 1 || t->pages < 1) return MARIAN_HIP_ERR_SHAPE;
  if(t->sequences > kMaxSequences || t->row > kMaxPositions / page || t->sequences * t->row > 0x7fffffff || t->pages > kMaxPositions / page)
    return MARIAN_HIP_ERR_RANGE;
  return MARIAN_HIP_OK;
}
// What a call on the tables writes (slots: null, or `slots_bytes`) shares no memory with anything else.
int check_tables_memory(const marian_hip_page_tables* t, const int32_t* lens, const int32_t* counts, int32_t* slots, int64_t slots_bytes) {
  if(!t->table || !t->held || !t->free || !t->free_count || !lens) return MARIAN_HIP_ERR_NULL;
  const void* all[7] = {t->table, t->held, t->free, t->free_count, lens, counts, slots};
  for(const void* p : all)
    if(!aligned(p, 4)) return MARIAN_HIP_ERR_ALIGN;
  const Span table{t->table, 4 * t->sequences * t->row}, held{t->held, 4 * t->sequences}, free{t->free, 4 * t->pages}, count{t->free_count, 4};
  const Span len{lens, 4 * t->sequences}, some{counts, 4 * t->sequences}, map{slots, slots_bytes};
  MH_CHECK(apart({table, held, free, count, map}, {len, some}));
  MH_CHECK(apart({table}, {held, free, count, map}));
  MH_CHECK(apart({held}, {free, count, map}));
  MH_CHECK(apart({free}, {count, map}));
  return apart({count}, {map});
}
TablesArgs tables_args(const marian_hip_page_tables* t, const int32_t* lens, const int32_t* counts, int64_t n, int64_t page, int32_t* slots) {
  TablesArgs a{};
  a.table = t->table;
  a.held = t->held;
  a.free = t->free;
  a.free_count = t->free_count;
  a.lens = lens;
  a.counts = counts;
  a.S = (int)t->sequences;
  a.row = (int)t->row;
  a.pages = (int)t->pages;
  a.n = (int)n;
  a.page = (int)page;
  a.by_page = CacheDivisor((unsigned)page);
  a.by_n = CacheDivisor((unsigned)std::max<int64_t>(n, 1));
  a.slots = slots;
  return a;
}

}  // namespace

extern "C" {

int marian_hip_pages_reserve(const marian_hip_page_tables* tables, const int32_t* lens, const int32_t* counts, int64_t n, int64_t page,
                             int32_t* slots, void* stream) {
  MH_CHECK(check_tables(tables, page));
  if(n < 0) return MARIAN_HIP_ERR_SHAPE;
  if(n > kMaxTokens || tables->sequences * n > 0x7fffffff) return MARIAN_HIP_ERR_RANGE;
  if(tables->sequences == 0 || n == 0) return MARIAN_HIP_OK;
  if(!slots) return MARIAN_HIP_ERR_NULL;
  MH_CHECK(check_tables_memory(tables, lens, counts, slots, 4 * tables->sequences * n));
  const TablesArgs a = tables_args(tables, lens, counts, n, page, slots);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  // One workgroup for up to eight slots a thread: 1024 sequences' two tokens 5.6 us, where two launches take some 9.
  const int64_t all = std::min<int64_t>(tables->sequences, kDealers) * n;   // (slots of one turn)
  if(tables->sequences * n <= 8 * kDealers) {
    MH_LAUNCH((pages_deal_kernel<false, true, true>), dim3(1), dim3(kDealers), 0, st, a);
    return MARIAN_HIP_OK;
  }
  MH_LAUNCH((pages_deal_kernel<false, true, false>), dim3((unsigned)std::min<int64_t>(256, (all + kDealers - 1) / kDealers)), dim3(kDealers), 0, st, a);
  MH_LAUNCH((pages_deal_kernel<false, false, true>), dim3(1), dim3(kDealers), 0, st, a);
  return MARIAN_HIP_OK;
}

int marian_hip_pages_trim(const marian_hip_page_tables* tables, const int32_t* lens, int64_t page, void* stream) {
  MH_CHECK(check_tables(tables, page));
  if(tables->sequences == 0) return MARIAN_HIP_OK;
  MH_CHECK(check_tables_memory(tables, lens, nullptr, nullptr, 0));
  const TablesArgs a = tables_args(tables, lens, nullptr, 0, page, nullptr);
  const hipStream_t st = static_cast<hipStream_t>(stream);
  // (how many pages go back only the device knows: the room for them stands for it)
  const int64_t moved = std::min(tables->sequences * tables->row, tables->pages);
  if(moved <= 4 * kDealers) {
    MH_LAUNCH((pages_deal_kernel<true, true, true>), dim3(1), dim3(kDealers), 0, st, a);
    return MARIAN_HIP_OK;
  }
  MH_LAUNCH((pages_deal_kernel<true, true, false>), dim3((unsigned)std::min<int64_t>(64, (std::min<int64_t>(tables->sequences, kDealers) + 15) / 16)), dim3(kDealers), 0, st, a);
  MH_LAUNCH((pages_deal_kernel<true, false, true>), dim3(1), dim3(kDealers), 0, st, a);
  return MARIAN_HIP_OK;
}

int marian_hip_pages_write(const marian_hip_pages* cache, const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                           int64_t sequences, int64_t n, const int32_t* slots, void* stream) {
  MH_CHECK(check_pages(cache));
  if(sequences < 0 || n < 0) return MARIAN_HIP_ERR_SHAPE;
  if(sequences > kMaxSequences || n > kMaxTokens) return MARIAN_HIP_ERR_RANGE;
  const int64_t row_bytes = cache->dk * width_of(cache->type), units = row_bytes / 16;
  if(sequences * n > (int64_t)0xffffff00 / (cache->heads * units)) return MARIAN_HIP_ERR_RANGE;
  if(sequences == 0 || n == 0) return MARIAN_HIP_OK;
  MH_CHECK(check_pages_memory(cache));
  if(!slots) return MARIAN_HIP_ERR_NULL;
  if(!aligned(slots, 4)) return MARIAN_HIP_ERR_ALIGN;
  Span ks, vs;
  MH_CHECK(check_rows(k, k_strides, cache->type, sequences, cache->heads, n, cache->dk, &ks));
  MH_CHECK(check_rows(v, v_strides, cache->type, sequences, cache->heads, n, cache->dk, &vs));
  const Span kp{cache->k, pages_bytes(cache)}, vp{cache->v, pages_bytes(cache)};
  MH_CHECK(apart({kp, vp}, {ks, vs, {slots, 4 * sequences * n}}));
  MH_CHECK(apart({kp}, {vp}));
  WriteArgs a{};
  a.k = static_cast<unsigned char*>(cache->k);
  a.v = static_cast<unsigned char*>(cache->v);
  a.kx = strides(k_strides);
  a.vx = strides(v_strides);
  a.slots = slots;
  a.heads = (int)cache->heads;
  a.page = (int)cache->page;
  a.row_bytes = (int)row_bytes;
  a.width = width_of(cache->type);
  a.pieces = (unsigned)(sequences * n * cache->heads * units);
  a.slots_end = (int)(cache->pages * cache->page);
  a.by_units = CacheDivisor((unsigned)units);
  a.by_heads = CacheDivisor((unsigned)cache->heads);
  a.by_n = CacheDivisor((unsigned)n);
  a.by_page = CacheDivisor((unsigned)cache->page);
  const unsigned each = 256 * kWriteTurns;
  const int64_t groups = ((int64_t)a.pieces + each - 1) / each;
  if(groups > kMostThreads / 256) return MARIAN_HIP_ERR_RANGE;
  MH_LAUNCH(pages_write_kernel, dim3((unsigned)groups), dim3(256), 0, static_cast<hipStream_t>(stream), static_cast<const unsigned char*>(k),
            static_cast<const unsigned char*>(v), a);
  return MARIAN_HIP_OK;
}

size_t marian_hip_pages_attention_workspace_bytes(int64_t sequences, int64_t heads, int64_t q_heads, int64_t n, int64_t dk, int type) {
  if(sequences < 1 || heads < 1 || q_heads < heads || q_heads % heads != 0 || n < 1 || !row_size(dk) || check_type(type) != MARIAN_HIP_OK) return 0;
  if(sequences > kMaxSequences || heads > kMaxHeads || q_heads / heads > kMaxHeads || n > kMaxTokens) return 0;
  return (size_t)pages_attention_bytes(pages_attention_plan(sequences, heads, q_heads, n, dk, width_of(type)), heads);
}

int marian_hip_pages_attention(const marian_hip_pages* cache, const int32_t* table, int64_t sequences, int64_t row, const int32_t* lens,
                               const int32_t* counts, int64_t n, const void* q, const int64_t* q_strides, int64_t q_heads, float scale, void* out,
                               const int64_t* out_strides, void* workspace, size_t workspace_bytes, void* stream) {
  MH_CHECK(check_pages(cache));
  const int64_t heads = cache->heads, dk = cache->dk, page = cache->page;
  const int type = cache->type, width = width_of(type);
  if(sequences < 0 || row < 1 || n < 0 || q_heads < heads || q_heads % heads != 0 || !(scale > 0.0f) || !std::isfinite(scale)) return MARIAN_HIP_ERR_SHAPE;
  if(sequences > kMaxSequences || row > kMaxPositions / page || sequences * row > 0x7fffffff || n > kMaxTokens || q_heads / heads > kMaxHeads ||
     n * (q_heads / heads) > 1 << 26)
    return MARIAN_HIP_ERR_RANGE;
  if(sequences == 0 || n == 0) return MARIAN_HIP_OK;
  const PagesAttentionPlan p = pages_attention_plan(sequences, heads, q_heads, n, dk, width, row * page);
  if(p.grid > kMostThreads / (64 * p.waves)) return MARIAN_HIP_ERR_RANGE;
  MH_CHECK(check_pages_memory(cache));
  if(!table || !lens) return MARIAN_HIP_ERR_NULL;
  if(!aligned(table, 4) || !aligned(lens, 4) || !aligned(counts, 4)) return MARIAN_HIP_ERR_ALIGN;
  Span qs, os;
  MH_CHECK(check_rows(q, q_strides, type, sequences, q_heads, n, dk, &qs));
  MH_CHECK(check_written(out, out_strides, type, sequences, q_heads, n, dk, &os));
  const int64_t need = pages_attention_bytes(p, heads);
  if(need > 0 && !workspace) return MARIAN_HIP_ERR_NULL;
  if((int64_t)workspace_bytes < need) return MARIAN_HIP_ERR_WORKSPACE;
  if(!aligned(workspace, 256)) return MARIAN_HIP_ERR_ALIGN;
  const Span work{need > 0 ? workspace : nullptr, need};
  MH_CHECK(apart({os, work}, {qs, {cache->k, pages_bytes(cache)}, {cache->v, pages_bytes(cache)}, {table, 4 * sequences * row}, {lens, 4 * sequences},
                              {counts, 4 * sequences}}));
  MH_CHECK(apart({os}, {work}));
  PagesAttentionArgs a{};
  a.q = q;
  a.q_s = q_strides[0];
  a.q_h = q_strides[1];
  a.q_n = q_strides[2];
  a.out = out;
  a.o_s = out_strides[0];
  a.o_h = out_strides[1];
  a.o_n = out_strides[2];
  a.lens = lens;
  a.counts = counts;
  a.counters = static_cast<unsigned*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + kCacheCounterBytes);
  a.S = (int)sequences;
  a.Hk = (int)heads;
  a.G = (int)(q_heads / heads);
  a.n = (int)n;
  a.cap = (int)(row * page);
  a.dk = (int)dk;
  a.row_tiles = (int)p.row_tiles;
  a.target = (int)p.target;
  a.least = p.least;
  a.items = (int)p.items;
  a.by_tiles = CacheDivisor((unsigned)p.row_tiles);
  a.by_heads = CacheDivisor((unsigned)heads);
  a.by_group = CacheDivisor((unsigned)a.G);
  a.scale_log2 = (float)((double)scale * 1.4426950408889634);
  a.k_pages = static_cast<const unsigned char*>(cache->k);
  a.v_pages = static_cast<const unsigned char*>(cache->v);
  a.table = table;
  a.row = (int)row;
  a.pages = (int)cache->pages;
  a.page = (int)page;
  a.head_bytes = page * dk * width;
  a.page_bytes = heads * a.head_bytes;
  a.by_eights = CacheDivisor((unsigned)(page / 8));
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if(type == MARIAN_HIP_FLOAT32) return launch_pages_attention_float32(a, p, st);
  if(type == MARIAN_HIP_FLOAT16) return launch_pages_attention_float16(a, p, st);
  return launch_pages_attention_bfloat16(a, p, st);
}

}  // extern "C"
