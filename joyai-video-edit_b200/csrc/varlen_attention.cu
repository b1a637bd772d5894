// Attention over requests of different lengths with grouped heads: new tokens
// over a paged K/V cache (paged_attention) and whole packed prompts
// (prompt_attention).  out = softmax(scale * q k^T) v over the visible keys,
// fp32 scores, statistics and accumulators, bf16 or fp16 in and out.
//
// Request b has the query rows query_starts[b] .. query_starts[b + 1] and
// kv_len keys; row i of its n rows sees keys 0 .. kv_len - n + i (causal) or
// all of them.  A row that sees no key is zero.
#include <math.h>

#include "jo_common.cuh"

namespace jo {
namespace vattn {

// What both forms share.  Strides in elements.
struct Params {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  const int32_t* starts;        // [batch + 1]
  const int32_t* kv_lens;       // [batch], NULL: as many keys as rows (packed prompts)
  const int32_t* table;         // [batch, width], NULL: keys packed like the queries
  int64_t q_ts, q_hs, k_bs, k_ts, k_hs, v_bs, v_ts, v_hs, o_ts, o_hs, table_stride;
  int tokens, batch, heads, group, head_dim, num_blocks, page, width, causal;
  float scale;
};

// Rows [first, first + n) and keys of request b; lengths are device data and
// are clamped to what the tensors hold.
struct Request {
  int first, n, keys;
};
__device__ __forceinline__ Request request(const Params& p, int b) {
  Request r;
  r.first = min(max(p.starts[b], 0), p.tokens);
  r.n = min(max(p.starts[b + 1], r.first), p.tokens) - r.first;
  r.keys = p.kv_lens ? (int)min((int64_t)max(p.kv_lens[b], 0), (int64_t)p.width * p.page) : r.n;
  return r;
}

// One warp per (token, head); D / 32 dimensions in each lane.
template <typename T, int D>
__global__ void __launch_bounds__(128) row_kernel(const Params p) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int t = (int)(w / p.heads), h = (int)(w - (int64_t)t * p.heads);
  if (t >= p.tokens) return;
  int a = 0, e = p.batch;
  while (e - a > 1) {
    const int mid = (a + e) >> 1;
    if (p.starts[mid] <= t) a = mid; else e = mid;
  }
  const Request r = request(p, a);
  if (t < r.first || t >= r.first + r.n) return;
  const int limit = p.causal ? max(0, r.keys - r.n + (t - r.first) + 1) : r.keys;
  const int hk = h / p.group;
  float q[E], o[E], m = -INFINITY, l = 0.f;
  for (int i = 0; i < E; ++i) {
    q[i] = to_f32(static_cast<const T*>(p.q)[t * p.q_ts + h * p.q_hs + lane * E + i]) * p.scale * 1.4426950408889634f;
    o[i] = 0.f;
  }
  for (int j = 0; j < limit; ++j) {
    int64_t kb, vb;
    bool in = true;
    if (p.table) {
      const int block = p.table[a * p.table_stride + j / p.page];
      in = block >= 0 && block < p.num_blocks;
      kb = block * p.k_bs + (j % p.page) * p.k_ts;
      vb = block * p.v_bs + (j % p.page) * p.v_ts;
    } else {
      kb = (r.first + j) * p.k_ts;
      vb = (r.first + j) * p.v_ts;
    }
    float s = 0.f, vv[E];
    for (int i = 0; i < E; ++i) {
      s = fmaf(q[i], in ? to_f32(static_cast<const T*>(p.k)[kb + hk * p.k_hs + lane * E + i]) : 0.f, s);
      vv[i] = in ? to_f32(static_cast<const T*>(p.v)[vb + hk * p.v_hs + lane * E + i]) : 0.f;
    }
    s = warp_sum(s);
    const float mn = fmaxf(m, s);
    const float al = exp2f(m - mn), pr = exp2f(s - mn);
    m = mn;
    l = l * al + pr;
    for (int i = 0; i < E; ++i) o[i] = o[i] * al + pr * vv[i];
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  for (int i = 0; i < E; ++i)
    static_cast<T*>(p.out)[t * p.o_ts + h * p.o_hs + lane * E + i] = from_f32<T>(o[i] * inv);
}

static int check(const char* what, Params& p, int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads,
                 int64_t head_dim, int dtype) {
  JO_REQUIRE(dtype == JO_DTYPE_BF16 || dtype == JO_DTYPE_F16, JO_ERR_DTYPE, "%s: only bf16 and fp16 are supported", what);
  JO_REQUIRE(head_dim == 64 || head_dim == 128, JO_ERR_INVALID, "%s: head_dim must be 64 or 128 (got %lld)", what,
             (long long)head_dim);
  JO_REQUIRE(tokens >= 0 && batch >= 0 && heads >= 0 && kv_heads >= 0 && tokens < (1LL << 30) && batch < (1LL << 30) &&
                 heads < 65536,
             JO_ERR_INVALID, "%s: invalid shape", what);
  JO_REQUIRE(heads == 0 || (kv_heads > 0 && heads % kv_heads == 0 && heads / kv_heads <= 128), JO_ERR_INVALID,
             "%s: heads (%lld) must be a multiple of kv_heads (%lld), at most 128 times it", what, (long long)heads,
             (long long)kv_heads);
  const int64_t s[10] = {p.q_ts, p.q_hs, p.k_bs, p.k_ts, p.k_hs, p.v_bs, p.v_ts, p.v_hs, p.o_ts, p.o_hs};
  for (int i = 0; i < 10; ++i)
    JO_REQUIRE(s[i] >= 0 && s[i] % 8 == 0, JO_ERR_ALIGN, "%s: strides must be non-negative multiples of 8 elements", what);
  JO_REQUIRE(aligned16(p.q) && aligned16(p.k) && aligned16(p.v) && aligned16(p.out), JO_ERR_ALIGN,
             "%s: tensors must be 16-byte aligned", what);
  p.tokens = (int)tokens;
  p.batch = (int)batch;
  p.heads = (int)heads;
  p.group = kv_heads > 0 ? (int)(heads / kv_heads) : 1;
  p.head_dim = (int)head_dim;
  return JO_OK;
}

static int launch(const char* what, const Params& p, int dtype, void* stream) {
  if (p.tokens == 0 || p.batch == 0 || p.heads == 0) return JO_OK;
  JO_REQUIRE(p.q && p.out && p.starts, JO_ERR_INVALID, "%s: null tensor pointer", what);
  int st = require_sm100();
  if (st != JO_OK) return st;
  const unsigned grid = (unsigned)(((int64_t)p.tokens * p.heads + 3) / 4);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == JO_DTYPE_BF16) {
    if (p.head_dim == 64) row_kernel<__nv_bfloat16, 64><<<grid, 128, 0, s>>>(p);
    else row_kernel<__nv_bfloat16, 128><<<grid, 128, 0, s>>>(p);
  } else {
    if (p.head_dim == 64) row_kernel<__half, 64><<<grid, 128, 0, s>>>(p);
    else row_kernel<__half, 128><<<grid, 128, 0, s>>>(p);
  }
  return check_launch(what);
}

}  // namespace vattn
}  // namespace jo

extern "C" {

int jo_paged_attention(const void* q, const void* key_cache, const void* value_cache, const int32_t* block_tables,
                       const int32_t* query_starts, const int32_t* kv_lens, void* out, int64_t tokens, int64_t batch,
                       int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t num_blocks, int64_t page_size,
                       int64_t table_width, int64_t table_stride, const int64_t* q_strides, const int64_t* kc_strides,
                       const int64_t* vc_strides, const int64_t* o_strides, int causal, float scale,
                       int64_t max_query_len, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace jo;
  const char* what = "paged_attention";
  JO_REQUIRE(q_strides && kc_strides && vc_strides && o_strides, JO_ERR_INVALID, "%s: null strides", what);
  JO_REQUIRE(page_size >= 16 && page_size % 16 == 0 && page_size < (1LL << 30), JO_ERR_INVALID,
             "%s: page_size must be a multiple of 16 (got %lld)", what, (long long)page_size);
  JO_REQUIRE(num_blocks >= 0 && num_blocks < (1LL << 31) && table_width >= 0 && table_width < (1LL << 31) &&
                 table_stride >= 0 && table_width * page_size < (1LL << 31),
             JO_ERR_INVALID, "%s: invalid cache or block table shape", what);
  vattn::Params p{q, key_cache, value_cache, out, query_starts, kv_lens, block_tables,
                  q_strides[0], q_strides[1], kc_strides[0], kc_strides[1], kc_strides[2],
                  vc_strides[0], vc_strides[1], vc_strides[2], o_strides[0], o_strides[1], table_stride};
  p.num_blocks = (int)num_blocks;
  p.page = (int)page_size;
  p.width = (int)table_width;
  p.causal = causal != 0;
  p.scale = scale;
  int st = vattn::check(what, p, tokens, batch, heads, kv_heads, head_dim, dtype);
  if (st != JO_OK) return st;
  JO_REQUIRE(tokens == 0 || batch == 0 || (kv_lens && block_tables && (num_blocks == 0 || (key_cache && value_cache))),
             JO_ERR_INVALID, "%s: null tensor pointer", what);
  return vattn::launch(what, p, dtype, stream);
}

int jo_prompt_attention(const void* q, const void* k, const void* v, const int32_t* seq_starts, void* out,
                        int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                        const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                        const int64_t* o_strides, int causal, float scale, int dtype, void* workspace,
                        int64_t workspace_bytes, void* stream) {
  using namespace jo;
  const char* what = "prompt_attention";
  JO_REQUIRE(q_strides && k_strides && v_strides && o_strides, JO_ERR_INVALID, "%s: null strides", what);
  vattn::Params p{q, k, v, out, seq_starts, nullptr, nullptr, q_strides[0], q_strides[1], 0, k_strides[0], k_strides[1],
                  0, v_strides[0], v_strides[1], o_strides[0], o_strides[1], 0};
  p.num_blocks = 0;
  p.page = 1;
  p.width = 0;
  p.causal = causal != 0;
  p.scale = scale;
  int st = vattn::check(what, p, tokens, batch, heads, kv_heads, head_dim, dtype);
  if (st != JO_OK) return st;
  JO_REQUIRE(tokens == 0 || batch == 0 || (k && v), JO_ERR_INVALID, "%s: null tensor pointer", what);
  return vattn::launch(what, p, dtype, stream);
}

int jo_varlen_attention_workspace(int64_t tokens, int64_t heads, int64_t head_dim, int64_t* bytes) {
  JO_REQUIRE(bytes, JO_ERR_INVALID, "varlen_attention_workspace: null pointer");
  (void)tokens, (void)heads, (void)head_dim;
  *bytes = 0;
  return JO_OK;
}

}  // extern "C"
