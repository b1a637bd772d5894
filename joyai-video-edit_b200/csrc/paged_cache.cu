// Block tables, slot maps and cache writes of a paged K/V cache.
//
// A cache is [num_blocks, page_size, kv_heads, head_dim]; request b holds the
// blocks block_tables[b, 0 ..], token position pos of it lives in slot
// block_tables[b, pos / page_size] * page_size + pos % page_size.
#include "jo_common.cuh"

namespace jo {
namespace paged {

constexpr int kThreads = 256;
constexpr int kPerThread = 4;                       // requests of one thread in a scan
constexpr int kChunk = kThreads * kPerThread;       // requests of one scan

using i64 = long long;

struct LayoutParams {
  const int32_t* cached;
  const int32_t* fresh;
  int32_t* table;
  const int32_t* free_blocks;
  int64_t batch, width, table_stride, num_free, tokens;
  uint32_t page;
  int32_t* starts;
  int32_t* kv_lens;
  int64_t* slots;
  int32_t* positions;
  int32_t* needed;
};

__device__ __forceinline__ int32_t saturate32(i64 v) {
  return (int32_t)(v > 0x7fffffffLL ? 0x7fffffffLL : v);
}

// Pages of n tokens (no n + page - 1, which may pass 32 bits).
__device__ __forceinline__ uint32_t pages(uint32_t n, uint32_t page) { return n / page + (n % page != 0); }

// Exclusive sums of (tokens, blocks) over the block's threads; the totals come
// back through `total`.  64 bits: lengths are device data and may add up to
// more than 31 bits.
__device__ __forceinline__ longlong2 block_scan(longlong2 v, longlong2* warp_sums, longlong2& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  longlong2 inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, inc.x, o), y = __shfl_up_sync(0xffffffffu, inc.y, o);
    if (lane >= o) inc.x += x, inc.y += y;
  }
  __syncthreads();  // the previous scan's sums have been read
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  longlong2 before = make_longlong2(0, 0);
  total = before;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) {
    const longlong2 s = warp_sums[w];
    if (w < warp) before.x += s.x, before.y += s.y;
    total.x += s.x, total.y += s.y;
  }
  return make_longlong2(before.x + inc.x - v.x, before.y + inc.y - v.y);
}

// One launch, no exchange between blocks.  Every block scans the request
// lengths (8 bytes each, from L2 after the first block) up to its own tokens
// and then looks its tokens' requests up by bisection; block 0 scans them all
// and writes the per-request outputs.  A page that a request newly needs
// starts at one of its new tokens, so the thread of that token writes the
// table entry, and a token's own slot follows from the free list without
// reading what another thread writes.  Latency-bound: a launch and a chain of
// a few dependent loads, whatever the sizes: 3.3 us for 48 requests of one token,
// 3.9 us for 300 requests and 25093 places, launch included.
__global__ void __launch_bounds__(kThreads) layout_kernel(const LayoutParams p) {
  __shared__ longlong2 warp_sums[kThreads / 32];
  __shared__ i64 s_start[kChunk];      // first token of the request
  __shared__ i64 s_base[kChunk];       // free blocks taken before the request
  __shared__ int32_t s_cached[kChunk];
  const i64 per_block = (p.tokens + gridDim.x - 1) / gridDim.x;
  const i64 t_begin = per_block * blockIdx.x;
  const i64 t_end = min(t_begin + per_block, (i64)p.tokens);
  const bool first = blockIdx.x == 0;
  i64 tok0 = 0, blk0 = 0;              // sums over the requests before this chunk
  for (i64 c0 = 0; c0 < p.batch && (first || tok0 < t_end); c0 += kChunk) {
    const int n = (int)min((i64)kChunk, (i64)p.batch - c0);
    i64 cached[kPerThread], fresh[kPerThread], need[kPerThread];
    longlong2 sum = make_longlong2(0, 0);
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int r = threadIdx.x * kPerThread + i;
      cached[i] = r < n ? max(0, p.cached[c0 + r]) : 0;
      fresh[i] = r < n ? max(0, p.fresh[c0 + r]) : 0;
      need[i] = (i64)pages((uint32_t)(cached[i] + fresh[i]), p.page) - pages((uint32_t)cached[i], p.page);
      sum.x += fresh[i];
      sum.y += need[i];
    }
    longlong2 total;
    longlong2 at = block_scan(sum, warp_sums, total);
    at.x += tok0;
    at.y += blk0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int r = threadIdx.x * kPerThread + i;
      if (r < n) {
        s_start[r] = at.x;
        s_base[r] = at.y;
        s_cached[r] = (int32_t)cached[i];
        if (first) {
          p.starts[c0 + r] = saturate32(at.x);
          p.kv_lens[c0 + r] = saturate32(cached[i] + fresh[i]);
        }
      }
      at.x += fresh[i];
      at.y += need[i];
    }
    __syncthreads();
    const i64 lo = max(t_begin, tok0), hi = min(t_end, tok0 + total.x);
    for (i64 t = lo + threadIdx.x; t < hi; t += kThreads) {
      int a = 0, b = n;                    // last request that starts at or before t
      while (b - a > 1) {
        const int mid = (a + b) >> 1;
        if (s_start[mid] <= t) a = mid; else b = mid;
      }
      const uint32_t old = (uint32_t)s_cached[a];
      const uint32_t pos = old + (uint32_t)(t - s_start[a]);
      const uint32_t j = pos / p.page, in_page = pos - j * p.page;
      const uint32_t held = pages(old, p.page);
      int32_t* entry = p.table + (c0 + a) * p.table_stride + j;
      int32_t block = -1;
      if (j < p.width) {
        if (j < held) {
          block = *entry;
        } else {
          const i64 f = s_base[a] + (j - held);
          if (f < p.num_free) block = p.free_blocks[f];
          if (in_page == 0) *entry = block;
        }
      }
      p.slots[t] = block >= 0 ? (i64)block * p.page + in_page : -1;
      p.positions[t] = (int32_t)pos;
    }
    __syncthreads();                       // the shared arrays are rewritten by the next chunk
    tok0 += total.x;
    blk0 += total.y;
  }
  // places after the last request (padding of a captured step)
  for (i64 t = max(t_begin, tok0) + threadIdx.x; t < t_end; t += kThreads) {
    p.slots[t] = -1;
    p.positions[t] = 0;
  }
  if (first && threadIdx.x == 0) {
    p.starts[p.batch] = saturate32(tok0);
    *p.needed = saturate32(blk0);
  }
}

struct WriteParams {
  const uint4* k;
  const uint4* v;
  uint4* kc;
  uint4* vc;
  const int64_t* slots;
  int64_t tokens, num_slots;
  uint32_t page, row_vecs, head_vecs;      // 16-byte vectors of a token and of a head
  // strides in vectors
  int64_t k_ts, k_hs, v_ts, v_hs, kc_bs, kc_ts, kc_hs, vc_bs, vc_ts, vc_hs;
};

// A thread takes the same 16-byte vector of K and of V of kTokens tokens, all loads before the first store: bound by HBM, and four
// loads in flight per thread keep it busy.  11042 tokens of 10 heads of 128: 20.0
// us, 5.65 TB/s (one token a thread 21.3 us, four 20.4).
constexpr int kTokens = 2;
__global__ void __launch_bounds__(kThreads) write_kernel(const WriteParams p) {
  const uint32_t x = blockIdx.y * blockDim.x + threadIdx.x;
  if (x >= p.row_vecs) return;
  const uint32_t h = x / p.head_vecs, d = x - h * p.head_vecs;
  const int64_t t0 = ((int64_t)blockIdx.x * blockDim.y + threadIdx.y) * kTokens;
  int64_t slot[kTokens];
  uint4 k[kTokens], v[kTokens];
#pragma unroll
  for (int i = 0; i < kTokens; ++i) slot[i] = t0 + i < p.tokens ? p.slots[t0 + i] : -1;
#pragma unroll
  for (int i = 0; i < kTokens; ++i)
    if (t0 + i < p.tokens) {
      k[i] = ld_stream(p.k + (t0 + i) * p.k_ts + h * p.k_hs + d);
      v[i] = ld_stream(p.v + (t0 + i) * p.v_ts + h * p.v_hs + d);
    }
#pragma unroll
  for (int i = 0; i < kTokens; ++i)
    if (slot[i] >= 0 && slot[i] < p.num_slots) {
      const int64_t block = slot[i] / p.page, in_page = slot[i] - block * p.page;
      p.kc[block * p.kc_bs + in_page * p.kc_ts + h * p.kc_hs + d] = k[i];
      p.vc[block * p.vc_bs + in_page * p.vc_ts + h * p.vc_hs + d] = v[i];
    }
}

}  // namespace paged
}  // namespace jo

extern "C" {

int jo_paged_layout(const int32_t* cached_lens, const int32_t* new_lens, int32_t* block_tables,
                    const int32_t* free_blocks, int64_t batch, int64_t table_width, int64_t table_stride,
                    int64_t num_free, int64_t page_size, int64_t num_tokens, int32_t* query_starts, int32_t* kv_lens,
                    int64_t* slots, int32_t* positions, int32_t* blocks_needed, void* stream) {
  using namespace jo;
  JO_REQUIRE(batch >= 0 && table_width >= 0 && num_free >= 0 && num_tokens >= 0 && batch < (1LL << 31) &&
                 num_tokens < (1LL << 31),
             JO_ERR_INVALID, "paged_layout: invalid shape");
  JO_REQUIRE(page_size >= 1 && page_size < (1LL << 30), JO_ERR_INVALID, "paged_layout: page_size must be positive");
  JO_REQUIRE(table_stride >= table_width || batch <= 1, JO_ERR_INVALID,
             "paged_layout: block table rows overlap (stride %lld, width %lld)", (long long)table_stride,
             (long long)table_width);
  JO_REQUIRE(query_starts && blocks_needed, JO_ERR_INVALID, "paged_layout: null output pointer");
  JO_REQUIRE(batch == 0 || (cached_lens && new_lens && kv_lens && (block_tables || table_width == 0)), JO_ERR_INVALID,
             "paged_layout: null tensor pointer");
  JO_REQUIRE(num_tokens == 0 || (slots && positions), JO_ERR_INVALID, "paged_layout: null output pointer");
  JO_REQUIRE(num_free == 0 || free_blocks, JO_ERR_INVALID, "paged_layout: null tensor pointer");
  int st = require_sm100();
  if (st != JO_OK) return st;
  paged::LayoutParams p{cached_lens, new_lens, block_tables, free_blocks, batch,     table_width, table_stride, num_free,
                        num_tokens,  (uint32_t)page_size, query_starts, kv_lens, slots, positions, blocks_needed};
  int64_t blocks = (num_tokens + paged::kThreads - 1) / paged::kThreads;
  blocks = blocks < 1 ? 1 : blocks > sm_count() ? sm_count() : blocks;
  paged::layout_kernel<<<(unsigned)blocks, paged::kThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return check_launch("paged_layout");
}

int jo_paged_kv_write(const void* key, const void* value, void* key_cache, void* value_cache, const int64_t* slots,
                      int64_t tokens, int64_t kv_heads, int64_t head_dim, int64_t num_blocks, int64_t page_size,
                      const int64_t* row_strides, const int64_t* cache_strides, int dtype, void* stream) {
  using namespace jo;
  JO_REQUIRE(dtype == JO_DTYPE_BF16 || dtype == JO_DTYPE_F16, JO_ERR_DTYPE, "paged_kv_write: only bf16 and fp16");
  JO_REQUIRE(tokens >= 0 && kv_heads >= 0 && num_blocks >= 0 && page_size >= 1 && tokens < (1LL << 31) &&
                 kv_heads < 65536 && num_blocks < (1LL << 31) && page_size < (1LL << 30),
             JO_ERR_INVALID, "paged_kv_write: invalid shape");
  JO_REQUIRE(head_dim >= 8 && head_dim % 8 == 0 && head_dim <= 65536, JO_ERR_INVALID,
             "paged_kv_write: head_dim must be a multiple of 8 (got %lld)", (long long)head_dim);
  if (tokens == 0 || kv_heads == 0 || num_blocks == 0) return JO_OK;
  JO_REQUIRE(key && value && key_cache && value_cache && slots && row_strides && cache_strides,
             JO_ERR_INVALID, "paged_kv_write: null pointer");
  int64_t all[10];
  for (int i = 0; i < 10; ++i) all[i] = i < 4 ? row_strides[i] : cache_strides[i - 4];
  // the stride of a dimension of one element is never used
  if (tokens == 1) all[0] = all[2] = 0;
  if (kv_heads == 1) all[1] = all[3] = all[6] = all[9] = 0;
  if (num_blocks == 1) all[4] = all[7] = 0;
  if (page_size == 1) all[5] = all[8] = 0;
  for (int i = 0; i < 10; ++i)
    JO_REQUIRE(all[i] >= 0 && all[i] % 8 == 0, JO_ERR_ALIGN,
               "paged_kv_write: strides must be non-negative multiples of 8 elements");
  JO_REQUIRE(aligned16(key) && aligned16(value) && aligned16(key_cache) && aligned16(value_cache), JO_ERR_ALIGN,
             "paged_kv_write: tensors must be 16-byte aligned");
  int st = require_sm100();
  if (st != JO_OK) return st;
  paged::WriteParams p;
  p.k = static_cast<const uint4*>(key);
  p.v = static_cast<const uint4*>(value);
  p.kc = static_cast<uint4*>(key_cache);
  p.vc = static_cast<uint4*>(value_cache);
  p.slots = slots;
  p.tokens = tokens;
  p.num_slots = num_blocks * page_size;
  p.page = (uint32_t)page_size;
  p.head_vecs = (uint32_t)(head_dim / 8);
  p.row_vecs = (uint32_t)(kv_heads * (head_dim / 8));
  int64_t* dst[10] = {&p.k_ts, &p.k_hs, &p.v_ts, &p.v_hs, &p.kc_bs, &p.kc_ts, &p.kc_hs, &p.vc_bs, &p.vc_ts, &p.vc_hs};
  for (int i = 0; i < 10; ++i) *dst[i] = all[i] / 8;
  // as many threads along a token's vectors as it has, up to a block's, and the rest along tokens
  unsigned bx = 32;
  while (bx < p.row_vecs && bx < (unsigned)paged::kThreads) bx *= 2;
  const unsigned by = paged::kThreads / bx;
  const int64_t gx = (tokens + by * paged::kTokens - 1) / (by * paged::kTokens);
  const int64_t gy = (p.row_vecs + bx - 1) / bx;
  JO_REQUIRE(gy < 65536, JO_ERR_INVALID, "paged_kv_write: too many elements in a token");
  paged::write_kernel<<<dim3((unsigned)gx, (unsigned)gy), dim3(bx, by), 0, static_cast<cudaStream_t>(stream)>>>(p);
  return check_launch("paged_kv_write");
}

}  // extern "C"
