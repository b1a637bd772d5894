// What the kernels of the variable-length attention share: the arguments, the
// division of the work over blocks, and the joining of partial results.
//
// An item is (request, key head, a run of the request's rows); its unit of work
// is one step over a fixed number of keys.  The units of all items, laid end to
// end in the order (request, key head, rows), are cut into one range per block,
// all of the same length, so that ragged lengths and single long requests fill
// the machine alike.  An item that a cut divides leaves partial results
// (maximum, sum, unnormalised rows), which join_kernel adds up in the order of
// the keys: results do not depend on timing.
#pragma once

#include "sm100_async.cuh"

namespace jo {
namespace vattn {

using namespace sm100;

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
  // Which requests a kernel takes, by their rows (tokens * group).
  int min_rows, max_rows;
};

// Rows [first, first + n) and keys of request b; n = 0 for one that this kernel
// does not take.  Lengths are device data and are clamped to what the tensors hold.
struct Request {
  int first, n, keys;
};
__device__ __forceinline__ Request request(const Params& p, int b) {
  Request r;
  r.first = min(max(p.starts[b], 0), p.tokens);
  r.n = min(max(p.starts[b + 1], r.first), p.tokens) - r.first;
  r.keys = p.kv_lens ? (int)min((long long)max(p.kv_lens[b], 0), (long long)p.width * p.page) : r.n;
  const long long rows = (long long)r.n * p.group;
  if (rows < p.min_rows || rows > p.max_rows) r.n = 0;
  return r;
}
// Keys that row i of the request sees.
__device__ __forceinline__ int visible(const Params& p, const Request& r, int i) {
  return p.causal ? max(0, r.keys - r.n + i + 1) : r.keys;
}

// Running maxima (of scale * log2(e) * s) start at the lowest finite number instead
// of at -infinity, so that a step in which a row sees no key leaves exp2(0) = 1 and
// exp2(-inf) = 0, and no NaN, while every finite score lies above it.
constexpr float kNoMax = -3.402823466e38f;

// A row's weights are exp2(x - m), where m = maximum - kUp and moves only when the
// maximum has grown by more than kLag since: the largest weight lies in 2^kUp ..
// 2^(kUp + kLag), and most steps leave the sums alone.  The weights are rounded to T
// before the product with V.  bf16 holds the small ones like the large ones.  fp16
// holds those below 2^-14 as multiples of 2^-24, so its weights are taken near the
// top of its range: multiples of 2^-35 of the largest (with the largest at 1, weights
// e^-14 and e^-16 were 0.35 and 5.9 % off, and a long tail of them with them).  It
// costs no time.
template <typename T> struct Weight { static constexpr float kUp = 0.f, kLag = 8.f; };
template <> struct Weight<__half> { static constexpr float kUp = 11.f, kLag = 4.f; };

__host__ __device__ __forceinline__ int div_up(int a, int b) { return (a + b - 1) / b; }

constexpr int kNear = 32;                // requests of a block's range that it keeps at hand

// floor(a / b) for 0 <= a < 2^52, b > 0.  Every block's first copy waits for a few
// of them: 32-bit divisions where the numbers allow, a 64-bit one takes hundreds
// of cycles.
__device__ __forceinline__ long long div_floor(long long a, long long b) {
  if (((a | b) >> 32) == 0) return (uint32_t)a / (uint32_t)b;
  long long q = (long long)((double)a / (double)b);
  if (q * b > a) --q;
  if ((q + 1) * b <= a) ++q;
  return q;
}

// KEYS keys of a step.  Beginning and ending an item costs as much as LEAD steps,
// which count as units of work too.  A cut closer than MIN steps to an item's edge
// moves to the edge: a shorter piece would cost more to join than to compute; and
// so does any cut in an item of at most WHOLE steps.
template <int KEYS, int LEAD, int MIN, int WHOLE>
struct Work {
  // Steps of item i: at least one, so that rows that see no key are written too.
  static __device__ __forceinline__ int steps(const Params& p, const Request& r, int i, int tpi) {
    const int last = min(r.n, (i + 1) * tpi) - 1;      // (rows are below 2^30, an item's tokens below 2^10)
    return max(1u, ((uint32_t)visible(p, r, last) + KEYS - 1) / KEYS);
  }

  // The even division of `total` units over `blocks` ranges.
  struct Cuts {
    long long total, each;               // the first `extra` ranges have one unit more than `each`
    int blocks, extra;
    __device__ __forceinline__ void divide(long long total_, int most) {
      total = total_;
      blocks = total >= (long long)most * (MIN + LEAD) ? most : max(1, (int)div_floor(total, MIN + LEAD));
      each = div_floor(total, blocks);
      extra = (int)(total - each * blocks);
    }
    __device__ __forceinline__ long long at(int c) const { return c >= blocks ? total : each * c + min(c, extra); }
    // the last range that begins at or before x
    __device__ __forceinline__ int of(long long x) const {
      const long long big = (each + 1) * extra;
      return x < big ? (int)div_floor(x, each + 1) : min(blocks - 1, extra + (int)div_floor(x - big, each));
    }
  };
  // Where a block's range lies.
  struct Range {
    int b, h, i, step;                   // its first step, which may be its item's end
    long long begin, end;                // units
    Cuts cuts;
  };
  // The range's requests, as far as they have room: every role of the block
  // walks over them, and a look at the lengths in global memory for each would
  // cost as much as a short request itself.
  struct Near {
    int count, next;                     // requests kept; where the ones after them begin
    int b[kNear];
    Request r[kNear];
  };
  struct Place {                         // a cut: the request it falls into and the units before it there
    int b, rank;
    long long off, per_head, at;
    Request r;
    int h, i, step;
  };
  template <int WARPS> struct Scan {
    longlong2 sums[WARPS];               // units, requests with rows
    Place cut[2];
  };

  // Units of one key head of a request, by one thread or by a warp.
  static __device__ __forceinline__ long long head_units(const Params& p, const Request& r, int tpi, int from, int by) {
    long long u = 0;
    for (int q = from; q * tpi < r.n; q += by) u += LEAD + steps(p, r, q, tpi);
    return u;
  }

  // Range of block c of at most C.  All threads of the block (WARPS warps) take
  // part, each looking after one request of a run of as many as there are threads.
  // Latency-bound: one look at the lengths (`early`: the one of the first run, asked
  // for as early as possible), a scan over the block, a few divisions.
  template <int WARPS>
  static __device__ void find(const Params& p, const Request& early, int tpi, int c, int C, Scan<WARPS>& s, Near& near,
                              Range& range) {
    constexpr int THREADS = 32 * WARPS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool one = p.batch <= THREADS; // one run holds them all
    Cuts cuts;
    long long begin = 0, end = 0;
    if (threadIdx.x < 2) s.cut[threadIdx.x] = Place{p.batch, 0, 0, 1, -1, {0, 0, 0}, 0, 0, 0};
    // First time round: the number of units, and where one run holds all the
    // cuts too.  Second: the cuts.
    for (int round = one ? 1 : 0; round < 2; ++round) {
      longlong2 base = make_longlong2(0, 0);
      for (int b0 = 0; b0 < p.batch; b0 += THREADS) {
        const int b = b0 + threadIdx.x;
        Request r = early;
        if (b0 > 0) r = b < p.batch ? request(p, b) : Request{0, 0, 0};
        long long u = 0;
        const bool many = r.n > 16 * tpi; // too many items for one thread
        if (!many) u = head_units(p, r, tpi, 0, 1);
        for (unsigned left = __ballot_sync(0xffffffffu, many); left; left &= left - 1) {
          const int src = __ffs(left) - 1;
          const Request w{0, __shfl_sync(0xffffffffu, r.n, src), __shfl_sync(0xffffffffu, r.keys, src)};
          long long v = head_units(p, w, tpi, lane, 32);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
          if (lane == src) u = v;
        }
        const longlong2 mine = make_longlong2(u * p.kv_heads, r.n > 0);
        longlong2 before = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const long long x = __shfl_up_sync(0xffffffffu, before.x, o), y = __shfl_up_sync(0xffffffffu, before.y, o);
          if (lane >= o) before.x += x, before.y += y;
        }
        __syncthreads();                 // the run before has been read
        if (lane == 31) s.sums[warp] = before;
        __syncthreads();
        before.x += base.x - mine.x;
        before.y += base.y - mine.y;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
          const longlong2 x = s.sums[w];
          if (w < warp) before.x += x.x, before.y += x.y;
          base.x += x.x, base.y += x.y;
        }
        if (round == 0) continue;
        if (one) {
          cuts.divide(base.x, C);
          begin = cuts.at(c);
          end = cuts.at(c + 1);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const long long t = k ? end : begin;
          if (t >= before.x && t < before.x + mine.x)
            s.cut[k] = Place{b, (int)before.y, t - before.x, u, t, r, 0, 0, 0};
        }
        if (one) {                       // this thread's request may be one of the range's
          __syncthreads();
          const int at = (int)before.y - s.cut[0].rank;
          if (r.n > 0 && b >= s.cut[0].b && b <= s.cut[1].b && at < kNear) {
            near.b[at] = b;
            near.r[at] = r;
          }
        }
      }
      if (round == 0) {
        cuts.divide(base.x, C);
        begin = cuts.at(c);
        end = cuts.at(c + 1);
      } else if (one && threadIdx.x == 0) {
        const int first = s.cut[0].b < p.batch ? s.cut[0].rank : (int)base.y;
        const int last = s.cut[1].b < p.batch ? s.cut[1].rank + 1 : (int)base.y;
        near.count = min(kNear, max(0, last - first));
      }
    }
    __syncthreads();
    // head, item and step of the two cuts, a warp for each
    if (warp < 2 && s.cut[warp].b < p.batch) {
      Place& f = s.cut[warp];
      const Request r = f.r;
      const int h = (int)div_floor(f.off, f.per_head);
      long long off = f.off - h * f.per_head;                // units into the key head's items
      for (int q0 = 0;; q0 += 32) {
        const int q = q0 + lane;
        const int n = q * tpi < r.n ? steps(p, r, q, tpi) : 0;
        int inc = n ? LEAD + n : 0;      // (32 items of at most 2^24 + LEAD units)
        const int u = inc;
        if (r.n > tpi) {
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += x;
          }
        }
        const unsigned hit = __ballot_sync(0xffffffffu, inc > off);
        if (hit) {
          if (lane == __ffs(hit) - 1) {
            long long step = off - (inc - u) - LEAD;
            if (step < MIN || (n <= WHOLE && 2 * step < n)) {
              f.at -= step + LEAD;
              step = 0;
            } else if (n - step < MIN || n <= WHOLE) {
              f.at += n - step;
              step = n;
            }
            f.h = h;
            f.i = q;
            f.step = (int)step;
          }
          break;
        }
        if (q0 + 32 >= r.n) break;       // (not reached: the cut lies in the request)
        off -= __shfl_sync(0xffffffffu, inc, 31);
      }
    }
    if (!one && warp == 2) {             // the range's requests, looked up again
      const int last = min(s.cut[1].b, p.batch - 1);
      int count = 0, b0 = s.cut[0].b;
      for (; b0 <= last && count < kNear; b0 += 32) {
        Request r{0, 0, 0};
        if (b0 + lane <= last) r = request(p, b0 + lane);
        const unsigned any = __ballot_sync(0xffffffffu, r.n > 0);
        const int at = count + __popc(any & ((1u << lane) - 1));
        if (r.n > 0 && at < kNear) {
          near.b[at] = b0 + lane;
          near.r[at] = r;
        }
        count += __popc(any);
      }
      if (lane == 0) near.count = min(count, kNear);
    }
    __syncthreads();
    if (threadIdx.x == 0) near.next = near.count > 0 ? near.b[near.count - 1] + 1 : p.batch;
    // a cut that falls into no request is the end of them all
    range = Range{s.cut[0].b, s.cut[0].h, s.cut[0].i, s.cut[0].step, s.cut[0].at < 0 ? cuts.total : s.cut[0].at,
                  s.cut[1].at < 0 ? cuts.total : s.cut[1].at, cuts};
  }

  // One block's stretch of one item.
  struct Piece {
    int b, h, i;
    Request r;
    int a, e;                            // steps [a, e) of the item's `steps`
    int steps;
    long long at;                        // unit at which the item's steps begin
    __device__ bool whole() const { return a == 0 && e == steps; }
  };

  // Walks a range piece by piece; every role of a block walks it for itself.
  struct Walk {
    const Params& p;
    const Near& near;
    int tpi, k, b, h, i, step;
    long long at, end;
    Request r;
    // (The range's first request is the first of the near ones: it has rows.)
    __device__ Walk(const Params& p_, int tpi_, const Near& near_, const Range& g)
        : p(p_), near(near_), tpi(tpi_), k(0), b(g.b), h(g.h), i(g.i), step(g.step), at(g.begin), end(g.end) {
      if (at < end) r = near.r[0];
    }
    __device__ void advance() {
      step = 0;
      if (++i * tpi < r.n) return;
      i = 0;
      if (++h < p.kv_heads) return;
      h = 0;
      if (++k < near.count) {
        b = near.b[k];
        r = near.r[k];
      } else {
        b = k == near.count ? near.next : b + 1;
        r.n = 0;
        for (; b < p.batch; ++b) {
          r = request(p, b);
          if (r.n > 0) break;
        }
        if (r.n == 0) at = end;
      }
    }
    __device__ bool next(Piece& s) {
      while (at < end) {
        const int n = Work::steps(p, r, i, tpi);
        if (step >= n) {
          advance();
          continue;
        }
        if (step == 0) at += LEAD;
        s.b = b;
        s.h = h;
        s.i = i;
        s.r = r;
        s.steps = n;
        s.a = step;
        s.e = (int)min((long long)n, step + max(1LL, end - at));
        s.at = at - step;
        at += s.e - s.a;
        if (at < end) advance();
        return true;
      }
      return false;
    }
  };

  // Blocks after this one that have a piece of the item that piece s begins: the
  // last of them begins before the item's end, and not so close to it that its
  // cut moved there.
  static __device__ int later_blocks(const Range& g, const Piece& s, int c) {
    return g.cuts.of(s.at + s.steps - MIN) - c;
  }
};

// ------------------------------------------------------- partial results ----
// Block c leaves at most two: slot 0 for an item that an earlier block began,
// slot 1 for one that later blocks go on with.
struct Begun {
  int later;     // blocks that go on with the item in slot 1; 0: no such item
  int first, n;  // its first row's token (absolute) and its tokens
  int h;
};
// R rows in column blocks of four, so that the rows of a warp are adjacent.
template <int D, int R> struct Slot {
  float o[D / 4][R][4];
  float2 ml[R];                          // maximum, sum
};

// Token and head of row r of an item whose rows come in tiles of TILE rows, tpt tokens each.
template <int TILE>
__device__ __forceinline__ bool row_place(int r, int group, int tpt, int n, int& tok, int& head) {
  const int t = r / TILE, in = r - t * TILE, k = in / group;
  tok = t * tpt + k;
  head = in - k * group;
  return k < tpt && tok < n;
}

// What one attention kernel left to join.
struct ToJoin {
  const void* slots;
  const Begun* begun;
  int blocks;                            // of the attention kernel
  int tpt;                               // tokens of a tile of rows
};

// Adds up the partial results of an item that cuts divide: the item that block c of
// the attention kernel began and did not end.  A team of TEAM warps takes 32 rows
// and 8 columns of it (y and the team's place in the block enumerate them), each
// lane one row; the team's warps share out the partial results and warp 0 adds
// theirs up.  Latency-bound: the reads of four partial results are in flight at a
// time.  Most blocks find nothing to do, and more or larger ones measured slower (54
// against 49 us for 64 single tokens over 54480 cached ones), fewer that look for
// work too (50.4).
// (Factors stop at kLeast, so that an infinity stays one however small its part.)
constexpr int kJoinWarps = 8;
constexpr float kLeast = 1.17549435e-38f;   // the smallest normal number
template <typename T, int D, int R, int TILE, int TEAM>
__device__ __forceinline__ void join_item(const Params& p, const ToJoin& j, int c, int y, float (*shared)[10][32]) {
  static_assert(kJoinWarps % TEAM == 0, "");
  const Slot<D, R>* slots = static_cast<const Slot<D, R>*>(j.slots);
  const Begun me = j.begun[c];
  if (me.later == 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, member = warp % TEAM;
  const int w = y * (kJoinWarps / TEAM) + warp / TEAM;
  const int col = (w % (D / 8)) * 8, r = (w / (D / 8)) * 32 + lane;
  int tok, head;
  const bool valid = row_place<TILE>(r, p.group, j.tpt, me.n, tok, head);
  float m = kNoMax, l = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  const int count = me.later + 1;        // slots 2c+1, 2c+2, 2c+4, ..., 2(c+later)
  const int per = (count + TEAM - 1) / TEAM, lo = member * per, hi = min(count, lo + per);
  constexpr int DEEP = 4;
  for (int i0 = lo; i0 < hi; i0 += DEEP) {
    float2 ml[DEEP];
    float4 x[DEEP], y[DEEP];
#pragma unroll
    for (int k = 0; k < DEEP; ++k) {
      const int i = min(i0 + k, hi - 1);
      const Slot<D, R>& s = slots[i == 0 ? 2 * c + 1 : 2 * (c + i)];
      ml[k] = s.ml[r];
      x[k] = *reinterpret_cast<const float4*>(s.o[col / 4][r]);
      y[k] = *reinterpret_cast<const float4*>(s.o[col / 4 + 1][r]);
    }
#pragma unroll
    for (int k = 0; k < DEEP; ++k) {
      if (i0 + k >= hi || ml[k].y == 0.f) continue;      // a row without a visible key there has no O either
      const float mn = fmaxf(m, ml[k].x), a = fmaxf(ex2(m - mn), kLeast), b = fmaxf(ex2(ml[k].x - mn), kLeast);
      m = mn;
      l = l * a + ml[k].y * b;
      const float v[8] = {x[k].x, x[k].y, x[k].z, x[k].w, y[k].x, y[k].y, y[k].z, y[k].w};
#pragma unroll
      for (int q = 0; q < 8; ++q) o[q] = o[q] * a + v[q] * b;
    }
  }
  if (TEAM > 1) {
    float(*mine)[32] = shared[warp];
    mine[0][lane] = m;
    mine[1][lane] = l;
#pragma unroll
    for (int q = 0; q < 8; ++q) mine[2 + q][lane] = o[q];
    __syncthreads();
    if (member != 0) return;
    for (int k = 1; k < TEAM; ++k) {
      float(*other)[32] = shared[warp + k];
      if (other[1][lane] == 0.f) continue;
      const float mo = other[0][lane], mn = fmaxf(m, mo), a = fmaxf(ex2(m - mn), kLeast), b = fmaxf(ex2(mo - mn), kLeast);
      m = mn;
      l = l * a + other[1][lane] * b;
#pragma unroll
      for (int q = 0; q < 8; ++q) o[q] = o[q] * a + other[2 + q][lane] * b;
    }
  }
  if (!valid) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint4 out;
  out.x = pack2<T>(o[0] * inv, o[1] * inv);
  out.y = pack2<T>(o[2] * inv, o[3] * inv);
  out.z = pack2<T>(o[4] * inv, o[5] * inv);
  out.w = pack2<T>(o[6] * inv, o[7] * inv);
  *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (int64_t)(me.first + tok) * p.o_ts +
                            (int64_t)(me.h * p.group + head) * p.o_hs + col) = out;
}
// Blocks along y that an item of R rows needs.
constexpr int join_y(int D, int R, int team) { return R / 32 * (D / 8) / (kJoinWarps / team); }

// ----------------------------------------------------------- K and V maps ----
// Byte of element (row, col) of a 128-byte-swizzled tile whose 64-column blocks
// are half_bytes apart.
__device__ __forceinline__ uint32_t swizzled(int row, int col, int half_bytes) {
  return (col >> 6) * half_bytes + row * 128 + ((((col & 63) * 2) >> 4 ^ (row & 7)) << 4) + ((col & 7) * 2);
}

// Maps of K and V for copies of `box` keys of one head: the largest power of two
// that divides the page, so that no copy crosses one, up to `most`.
inline bool kv_maps(const Params& p, bool bf16, int most, CUtensorMap* k, CUtensorMap* v, int* box) {
  if (p.table) {
    *box = p.page & -p.page;
    if (*box > most) *box = most;
    const int kb[4] = {64, 1, *box, 1};
    // an empty cache: every block is outside it, the address is never read
    const int64_t d[4] = {p.head_dim, p.kv_heads, p.page, p.num_blocks > 0 ? p.num_blocks : 1};
    const int64_t ks[3] = {p.k_hs, p.k_ts, p.k_bs}, vs[3] = {p.v_hs, p.v_ts, p.v_bs};
    return make_map_4d(k, bf16, p.num_blocks > 0 ? p.k : p.q, d, ks, kb) &&
           make_map_4d(v, bf16, p.num_blocks > 0 ? p.v : p.q, d, vs, kb);
  }
  *box = most;
  const int kb[4] = {64, 1, most, 1};
  const int64_t d[4] = {p.head_dim, p.kv_heads, p.tokens, 1};
  const int64_t ks[3] = {p.k_hs, p.k_ts, 0}, vs[3] = {p.v_hs, p.v_ts, 0};
  return make_map_4d(k, bf16, p.k, d, ks, kb) && make_map_4d(v, bf16, p.v, d, vs, kb);
}

// Coordinates (z, w) of key `key` of request b in those maps; a block outside the
// cache, and a key past the request's, read as zeros.  first: the row of its first
// key where keys are packed.
__device__ __forceinline__ void kv_place(const Params& p, int first, int keys, int b, int key, int& z, int& w) {
  if (p.table) {
    const int pg = key / p.page;
    z = key - pg * p.page;
    int block = -1;
    if (key < keys) block = p.table[(int64_t)b * p.table_stride + pg];
    w = block >= 0 && block < p.num_blocks ? block : -1;
  } else {
    z = first + key;
    w = 0;
  }
}

// ---------------------------------------------------- infinite values of V ----
// An infinity in V that a row sees makes its result infinite, but in the products
// a weight (or the rest of one) that rounds to zero turns it into NaN.  V is not searched
// for them on the way: a piece whose sums hold a NaN, though its weights are
// numbers, looks through the keys again when it ends and takes from there what its
// columns see.  So only calls that meet infinities or NaN pay for it (the look at
// the sums: 8.1 us before and after at one short request, at most 0.3 of 49 us at
// 64 single tokens).
//
// V of one key head of a request, in global memory.
struct Values {
  const void* v;
  const int32_t* table;                  // the request's row, NULL: keys packed
  int64_t block_stride, key_stride;      // elements
  int page, num_blocks;
  __device__ Values(const Params& p, int first, int b, int h) {
    table = p.table ? p.table + (int64_t)b * p.table_stride : nullptr;
    v = static_cast<const uint16_t*>(p.v) + (int64_t)h * p.v_hs + (p.table ? 0 : (int64_t)first * p.v_ts);
    block_stride = p.v_bs;
    key_stride = p.v_ts;
    page = p.page;
    num_blocks = p.num_blocks;
  }
  // 8 columns of a key (below the request's keys)
  __device__ __forceinline__ uint4 at(int key, int col) const {
    int64_t place = (int64_t)key * key_stride;
    if (table) {
      const int pg = key / page, block = table[pg];
      if (block < 0 || block >= num_blocks) return make_uint4(0, 0, 0, 0);
      place = (int64_t)block * block_stride + (int64_t)(key - pg * page) * key_stride;
    }
    return *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(v) + place + col);
  }
};

template <typename T> __device__ __forceinline__ void add_odd(float (&sum)[8], uint4 x) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t bits = (i & 1 ? w[i >> 1] >> 16 : w[i >> 1]) & 0xffffu;
    if ((bits & 0x7fffu) >= Bits16<T>::kInf) sum[i] += from_bits16<T>(bits);
  }
}

// out[i] = sum of the values in column col + i that are not finite (0: there are
// none) among the keys [from, min(to, limit)) of this lane's row, for the columns
// whose bit is set in `need` of any lane.  A whole warp calls it with rows that all
// see the keys below `common`, and shares those out, until every such column has met
// a NaN.
template <typename T>
__device__ __noinline__ void odd_values(const Values v, int col, uint32_t need, int from, int common, int to, int limit,
                                        float* out) {
  const int lane = threadIdx.x & 31;
  float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  need = __reduce_or_sync(0xffffffffu, need);
  common = min(common, to);
  bool more = need != 0;
  for (int key0 = from; more && key0 < common; key0 += 256) {
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (key0 + 32 * k + lane < common) add_odd<T>(sum, v.at(key0 + 32 * k + lane, col));
    uint32_t nan = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) nan |= (sum[i] != sum[i] ? 1u : 0u) << i;
    more = (need & ~__reduce_or_sync(0xffffffffu, nan)) != 0;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
  if (more)
#pragma unroll 1
    for (int key = max(from, common); key < min(to, limit); ++key) add_odd<T>(sum, v.at(key, col));
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) out[i] = sum[i];
}
// What a sum becomes: `odd` of its column.  total: the row's sum of weights (NaN where
// a weight is one, 0 where it sees no key).
__device__ __forceinline__ bool is_odd(float sum, float total) { return sum != sum && total > 0.f; }
__device__ __forceinline__ float with_odd(float sum, float odd, float total) {
  return is_odd(sum, total) && odd != 0.f ? odd : sum;
}

// The kernel for requests of few rows (varlen_few.cu): `rows`, the most of any
// request as far as the host knows; up to kFewRows it serves them best.  What is
// to be joined comes back in *join (blocks 0: nothing).  beside: its blocks may
// begin as those of the kernel before it end, of which it needs nothing.
constexpr int kFewRows = 32;
struct FewShape {
  int rows16;                            // rows of an item / 16: 1 or 2
};
int64_t few_workspace(int head_dim);
bool few_splits(int64_t max_keys);       // whether an item of so many keys can have a cut inside
int launch_few(const char* what, const Params& p, int64_t rows, int dtype, void* workspace, bool beside, ToJoin* join,
               FewShape* shape, cudaStream_t stream);
int few_last_fault(int reset);

}  // namespace vattn
}  // namespace jo
