// What the kernels of the variable-length attention share: the arguments, the
// requests' lengths, and the partial results of work that is split along the keys.
#pragma once

#include "jo_common.cuh"

namespace jo {
namespace vattn {

// Strides in elements.
struct Params {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  const int32_t* starts;        // [batch + 1]
  const int32_t* kv_lens;       // [batch], NULL: as many keys as rows (packed prompts)
  const int32_t* table;         // [batch, width], NULL: keys packed like the queries
  int64_t q_ts, q_hs, k_bs, k_ts, k_hs, v_bs, v_ts, v_hs, o_ts, o_hs, table_stride;
  int tokens, batch, heads, kv_heads, group, head_dim, num_blocks, page, width, causal;
  float scale_log2;             // |scale| * log2(e), never 0
  int negate;                   // scale < 0
};

// Rows [first, first + n) and keys of request b.  Lengths are device data and
// are clamped to what the tensors hold.
struct Request {
  int first, n, keys;
};
__device__ __forceinline__ Request request(const Params& p, int b) {
  Request r;
  r.first = min(max(p.starts[b], 0), p.tokens);
  r.n = min(max(p.starts[b + 1], r.first), p.tokens) - r.first;
  r.keys = p.kv_lens ? (int)min((long long)max(p.kv_lens[b], 0), (long long)p.width * p.page) : r.n;
  return r;
}
// Keys that row i of the request sees.
__device__ __forceinline__ int visible(const Params& p, const Request& r, int i) {
  return p.causal ? max(0, r.keys - r.n + i + 1) : r.keys;
}

// Running maxima (of scale * log2(e) * s) start here instead of at -infinity, so
// that a tile in which a row sees no key leaves exp2(0) = 1 and exp2(-inf) = 0,
// and no NaN.
constexpr float kNoMax = -1e30f;

}  // namespace vattn
}  // namespace jo
