// Attention over requests of different lengths with grouped heads: new tokens
// over a paged K/V cache (paged_attention) and whole packed prompts
// (prompt_attention).  out = softmax(scale * q k^T) v over the visible keys,
// fp32 scores, statistics and accumulators, bf16 or fp16 in and out.
//
// Request b has the query rows query_starts[b] .. query_starts[b + 1] and
// kv_len keys; row i of its n rows sees keys 0 .. kv_len - n + i (causal) or
// all of them.  A row that sees no key, or only scores of -infinity, is zero.
//
// Organisation of tile_kernel (one block per SM, 384 threads).  The `group`
// query heads that read one key head are rows of one tile: row r of a tile is
// token r / group, head r % group, so K and V are read once for all of them.
// An item is (request, key head, 256 rows as two 128-row tiles), a step 128 keys;
// the steps of all items are shared out evenly (varlen_attention.cuh).
//   warp 8       TMA producer: Q tiles of an item, K and V of every step (pages
//                looked up in the block table, one copy per run of a page)
//   warp 9       MMA issuer: S_t = Q_t K^T, O_t += P_t V on tcgen05, in the order
//                PV0 QK0' PV1 QK1' so that the softmax of one tile overlaps the
//                MMAs of the other, across items too
//   warp 10      looks after V in steps where some row does not see every key:
//                rows past the last visible key are zeroed (a product with P = 0
//                would turn a NaN there into NaN), and a value row that only some
//                rows may see is searched for NaN and infinities
//   warp 11      walks the block's range and hands its pieces to the others
//
// PAIR: two blocks (a cluster) take an item of 512 rows together, tile t of the
// one above tile t of the other in one cta_group::2 MMA of 256 rows.  Each block
// loads half of K's keys and half of V's columns, so the shared memory that an MMA
// reads besides its own 128 rows, what bounds it in the single form, is halved, and
// twice as many steps are in flight.  The even block issues the MMAs.
//   warps 0-7    softmax: one thread per row, P over S in tensor memory
// The weights' reference only moves when the maximum has grown enough, so most steps
// leave O alone.  They are rounded once to the tensors' type, as the matrix
// instruction takes them: a second product for the rest, as in varlen_few.cu, would
// double PV.  Results have 1.1-1.4 times the error of rounding them alone.
//
// What bounds it: for long requests the chain of a tile, softmax (1750 cycles), P
// seen by the MMA warp (450), PV and the next QK into the place that P leaves
// (1240), S seen (250), of which two tiles fill 2480 of 3900 cycles on the tensor
// cores; then the power limit.  One causal prompt of 12288 tokens, 16 heads over 4
// of 128: 557-650 us, 0.95-1.11 PFLOP/s by the clocks that the limit leaves; 11042
// tokens over 32102 keys, 10 heads: 1.70-1.92 ms, 0.95-1.07 PFLOP/s.  For short ones
// dependent round trips: lengths, division of the work, block table, first scores 5
// us after the start, 4-5 us for an item of one step.
#include <math.h>

#include "varlen_attention.cuh"

namespace jo {
namespace vattn {

constexpr int kRows = 128;               // rows of a tile
constexpr int kKeys = 128;               // keys of a step
constexpr int kThreads = 384;
// Blocks work in pairs where requests have this many rows and K and V may be larger
// than L2 by half: the host knows what the tables and the cache can hold, not the
// lengths (kv_bytes).  Pairs halve the reads of K and V and have twice the steps in
// flight, but wait for each other.  Single form and pairs, measured in turn: 11042
// tokens over 32102 keys, 20 heads (K and V 329 MB) 4.05 and 3.57 ms, 10 heads (164
// MB) 1.83 and 1.72 in one run, 1.00-1.08 and 1.00 PFLOP/s in another; 10 heads,
// 2048 tokens over 10048 keys 115 and 118 us, over 2548 47 and 52 us, which is what a
// chunk over a short history costs more where tables and cache are large.
constexpr int kPairRows = 2048;
constexpr int64_t kPairBytes = 192LL << 20;
// Steps that an item's beginning and end cost; steps of the shortest piece; items
// that are never cut.  (Beginnings at 1, 3, 4, pieces of 1, 3, 4: ragged prompts
// 212-234 us against 209, mixed chunks 52-57 against 53.)
constexpr int kLead = 2, kMin = 2, kWhole = 3;
using Steps = Work<kKeys, kLead, kMin, kWhole>;
using Range = Steps::Range;
using Piece = Steps::Piece;
using Walk = Steps::Walk;

__device__ int g_fault = 0;

constexpr int kPieces = 8;               // pieces handed out ahead

// A piece as the roles need it.
struct Task {
  int a, e;                              // steps [a, e); e < 0: the range's end
  int end[2];                            // tile t takes part in steps [a, end[t])
  int edge;                              // first step in which some row does not see every key
  int tok, ntok;                         // the item's first token (absolute) and its tokens
  int before;                            // keys before its first token (causal: token k sees before + k + 1)
  int keys, kfirst;                      // the request's keys, and their first row where they are packed
  int b, h;
  int slot;                              // -1: the piece is a whole item, else the slot of its partial result
  int pad[3];
};

template <int D, bool PAIR> struct Cfg {
  static constexpr int N = PAIR ? 2 : 1;                     // blocks of an item
  static constexpr int HALVES = D / 64;
  static constexpr int HALF = kRows * 128;                   // 128 rows x 64 elements
  static constexpr int TILE = HALVES * HALF;                 // Q
  static constexpr int STAGE = TILE / N;                     // this block's part of K or V of a step
  static constexpr int KHALF = HALF / N;                     // K: its keys x 64 elements
  static constexpr int ST = 65536 / STAGE;                   // K and V steps in flight, 64 KB each
  static constexpr int K0 = 2 * TILE, V0 = K0 + ST * STAGE;
  static constexpr int OUT = V0 + ST * STAGE;                // 2 KB of a softmax warp: 32 rows x 32 columns on their way out
  static constexpr int TASKS = OUT + 8 * 2048;
  static constexpr int BARS = TASKS + kPieces * (int)sizeof(Task);
  enum : int { B_QF = 0, B_QE = 1, B_SF = 2, B_PF = 4, B_OF = 6, B_TF = 8, B_TE = B_TF + kPieces, B_KF = B_TE + kPieces,
               B_KE = B_KF + ST, B_VF = B_KE + ST, B_VE = B_VF + ST, B_VG = B_VE + ST, B_END = B_VG + ST, B_N };
  static constexpr int BYTES = BARS + 512 /* barriers, flags */ + 1024 /* alignment */;
  static_assert(B_N * 8 + 8 + 4 * N * ST <= 512, "");
  static_assert(!PAIR || D == 128, "");
};

struct Maps {
  CUtensorMap q, k, v;
  int tpt;                               // tokens of a tile: 128 / group
  int box;                               // keys of one K or V copy
  void* partial;
  Begun* begun;
};

// Keys that token k of the task's item sees.
__device__ __forceinline__ int task_visible(const Params& p, const Task& t, int k) {
  return p.causal ? max(0, t.before + k + 1) : t.keys;
}

// O (+)= P V for one row on the CUDA cores: the step's V holds a NaN or an
// infinity that this row may not see, and a matrix product would spread it.
// v0, v1: cluster addresses of the step's V, columns 0-63 and 64-127.
template <typename T, int D>
__device__ __noinline__ void careful_pv(uint32_t tP, uint32_t tO, uint32_t v0, uint32_t v1, bool first, int lim) {
#pragma unroll 1
  for (int c = 0; c < D; c += 32) {
    uint32_t o[32];
    if (first) {
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] = 0u;
    } else {
      tmem_ld32(tO + c, o);
      tmem_wait_ld();
    }
#pragma unroll 1
    for (int k = 0; k < kKeys; k += 16) {
      uint32_t pw[8];
      tmem_ld8(tP + k / 2, pw);
      tmem_wait_ld();
#pragma unroll 1
      for (int kk = 0; kk < 16; ++kk) {
        uint32_t word = pw[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) word = (kk >> 1) == i ? pw[i] : word;
        const float2 pp = unpack2<T>(word);
        const float pj = kk & 1 ? pp.y : pp.x;
        const bool seen = k + kk < lim;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 x = ld_cluster((c < 64 ? v0 : v1) + swizzled(k + kk, (c & 63) + 8 * i, 0));
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float2 f = unpack2<T>(w[q]);
            const int at = 8 * i + 2 * q;
            if (seen) {
              o[at] = __float_as_uint(fmaf(pj, f.x, __uint_as_float(o[at])));
              o[at + 1] = __float_as_uint(fmaf(pj, f.y, __uint_as_float(o[at + 1])));
            }
          }
        }
      }
    }
    tmem_st32(tO + c, o);
  }
  tmem_wait_st();
}

// Puts into 32 columns of O in tensor memory, from col, the infinities that this
// lane's row sees in V (varlen_attention.cuh).
template <typename T>
__device__ __noinline__ void repair_odd(const Values v, uint32_t tO, int col, int from, int to, int limit, float total) {
  const int common = __reduce_min_sync(0xffffffffu, limit);
  uint32_t o[32];
  tmem_ld32(tO, o);
  tmem_wait_ld();
#pragma unroll
  for (int c = 0; c < 32; c += 8) {
    uint32_t need = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) need |= (is_odd(__uint_as_float(o[c + i]), total) ? 1u : 0u) << i;
    float x[8];
    odd_values<T>(v, col + c, need, from, common, to, limit, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[c + i] = __float_as_uint(with_odd(__uint_as_float(o[c + i]), x[i], total));
  }
  tmem_st32(tO, o);
  tmem_wait_st();
}

template <typename T, int D, bool PAIR>
__global__ void __launch_bounds__(kThreads, 1) tile_kernel(const __grid_constant__ Maps maps, const Params p) {
  using C = Cfg<D, PAIR>;
  constexpr int ST = C::ST, N = C::N;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  __shared__ Steps::Scan<kThreads / 32> scan;
  __shared__ Steps::Near near;
  unsigned char* smem =
      reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  Task* tasks = reinterpret_cast<Task*>(smem + C::TASKS);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::BARS);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::B_N);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  volatile int* vflag = abort_flag + 1;  // [ST][N]: a NaN or infinity found in an edge step's V, by each block's guard
  const uint32_t bar0 = smem_u32(bars);
#define BAR(i) (bar0 + 8u * (uint32_t)(i))
#define WAIT(i, parity, code) mbar_wait(BAR(i), (parity), abort_flag, &g_fault, (code))
// The next task of a role that has had n of them.
#define NEXT_TASK(n) (WAIT(C::B_TF + (n) % kPieces, ((n) / kPieces) & 1, 20))
#define TASK(n) (tasks[(n) % kPieces])

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = PAIR ? cluster_rank() : 0;
  const int unit = blockIdx.x / N;       // the block or pair among its like
  wait_for_primary();                    // launched as the kernel before it ends
  const Request early = (int)threadIdx.x < p.batch ? request(p, threadIdx.x) : Request{0, 0, 0};
  launch_dependents();
  if (threadIdx.x == 0) {
    mbar_init(BAR(C::B_QF), 1);
    mbar_init(BAR(C::B_QE), 1);
    mbar_init(BAR(C::B_END), 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(BAR(C::B_SF + t), 1);
      mbar_init(BAR(C::B_PF + t), 4 * N);          // one arrival per softmax warp (on the even block's)
      mbar_init(BAR(C::B_OF + t), 1);
    }
    for (int s = 0; s < kPieces; ++s) {
      mbar_init(BAR(C::B_TF + s), 1);
      mbar_init(BAR(C::B_TE + s), rank == 0 ? 11 : 10);   // every warp but the one that hands them out; one issues MMAs
    }
    for (int s = 0; s < ST; ++s) {
      mbar_init(BAR(C::B_KF + s), 1);
      mbar_init(BAR(C::B_KE + s), 1);
      mbar_init(BAR(C::B_VF + s), 1);
      mbar_init(BAR(C::B_VE + s), 1);
      mbar_init(BAR(C::B_VG + s), N);              // one per guard
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
  }
  if (warp == 8 && lane == 0) {
    tma_prefetch_map(&maps.q);
    tma_prefetch_map(&maps.k);
    tma_prefetch_map(&maps.v);
  }
  if (warp == 9) tmem_alloc_512<PAIR>(smem_u32(tmem_slot));
  Range range;
  Steps::find<kThreads / 32>(p, early, 2 * N * maps.tpt, unit, gridDim.x / N, scan, near, range);
  fence_before();
  if (PAIR) cluster_sync(); else __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t sq = smem_u32(smem), sk = sq + C::K0, sv = sq + C::V0;
  const int tpt = maps.tpt;
  // place `bar` in the even block
  auto even = [&](uint32_t bar) { return PAIR ? map_to_rank(bar, 0) : bar; };

  if (warp == 11) {
    // ------------------------------------------------------ hands out pieces --
    if (lane == 0) {
      Walk walk(p, 2 * N * tpt, near, range);
      Piece s;
      Begun begun{0, 0, 0, 0};
      bool more = true;
      for (uint32_t n = 0; more; ++n) {
        if (!WAIT(C::B_TE + n % kPieces, ((n / kPieces) & 1) ^ 1, 21)) {
          begun.later = 0;
          break;
        }
        more = walk.next(s);
        Task t;
        t.a = 0;
        t.e = -1;
        if (more) {
          const int tok = s.i * 2 * N * tpt;
          t.a = s.a;
          t.e = s.e;
          t.tok = s.r.first + tok;
          t.ntok = min(2 * N * tpt, s.r.n - tok);
          t.before = s.r.keys - s.r.n + tok;
          t.keys = s.r.keys;
          t.kfirst = s.r.first;
          t.b = s.b;
          t.h = s.h;
          t.edge = (uint32_t)task_visible(p, t, 0) / kKeys;
          t.end[0] = max(s.a, min(s.e, (int)max(1u, ((uint32_t)task_visible(p, t, min(t.ntok, N * tpt) - 1) + kKeys - 1) / kKeys)));
          t.end[1] = t.ntok > N * tpt ? s.e : s.a;
          t.slot = s.whole() ? -1 : 2 * unit + (s.a == 0 ? 1 : 0);
          if (s.a == 0 && s.e < s.steps)       // only the last piece ends inside an item
            begun = Begun{Steps::later_blocks(range, s, unit), t.tok, t.ntok, t.h};
        }
        TASK(n) = t;
        mbar_arrive(BAR(C::B_TF + n % kPieces));
      }
      if (maps.begun && rank == 0) maps.begun[unit] = begun;
    }
  } else if (warp == 8) {
    // ------------------------------------------------------------- producer --
    // This lane's copies of a step: `box` keys x 64 columns of K and of V each.
    // A pair's block has half of K's keys and half of V's columns.
    const int copies = kKeys / maps.box * C::HALVES / N;
    const bool mine = lane < copies;
    const int k_boxes = kKeys / N / maps.box, v_boxes = kKeys / maps.box;
    const int kb = lane % k_boxes, kh = lane / k_boxes, vb = lane % v_boxes, vh = lane / v_boxes;
    const int k_key = rank * (kKeys / 2) + kb * maps.box, v_key = vb * maps.box;
    const uint32_t k_dst = kh * C::KHALF + kb * maps.box * 128, v_dst = vh * C::HALF + vb * maps.box * 128;
    const int k_col = kh * 64, v_col = (PAIR ? rank : vh) * 64;
    uint32_t it = 0, v_issued = 0, n = 0;
    for (;; ++n) {
      if (!__all_sync(0xffffffffu, NEXT_TASK(n))) break;
      const Task t = TASK(n);
      __syncwarp();
      if (lane == 0) mbar_arrive(BAR(C::B_TE + n % kPieces));
      if (t.e < 0) break;
      // Places of 16 keys each (pages are multiples of 16 keys), four steps at a
      // time; those of the next four are looked up meanwhile.
      int z0 = 0, w0 = 0, z1, w1;
      kv_place(p, t.kfirst, t.keys, t.b, t.a * kKeys + lane * 16, z1, w1);
      bool ok = true;
      for (int j = t.a; j < t.e; ++j, ++it) {
        const int ahead = (j - t.a) & 3;
        if (ahead == 0) {
          z0 = z1;
          w0 = w1;
          kv_place(p, t.kfirst, t.keys, t.b, (j + 4) * kKeys + lane * 16, z1, w1);
        }
        const int k_from = (ahead * 8 + k_key / 16) & 31, v_from = (ahead * 8 + v_key / 16) & 31;
        const int kz = __shfl_sync(0xffffffffu, z0, k_from), kw = __shfl_sync(0xffffffffu, w0, k_from);
        const int vz = __shfl_sync(0xffffffffu, z0, v_from), vw = __shfl_sync(0xffffffffu, w0, v_from);
        const int st = it % ST;
        const uint32_t ph = (it / ST) & 1;
        ok = __all_sync(0xffffffffu, WAIT(C::B_KE + st, ph ^ 1, 1));
        if (!ok) break;
        // K's and Q's completion is counted on the even block's barriers, for both
        if (lane == 0 && rank == 0) mbar_expect_tx(BAR(C::B_KF + st), N * C::STAGE);
        __syncwarp();
        if (mine) {
          if (PAIR) tma_load_4d_pair(sk + st * C::STAGE + k_dst, &maps.k, k_col, t.h, kz, kw, even(BAR(C::B_KF + st)));
          else tma_load_4d(sk + st * C::STAGE + k_dst, &maps.k, k_col, t.h, kz, kw, BAR(C::B_KF + st));
        }
        if (j == t.a) {
          ok = __all_sync(0xffffffffu, WAIT(C::B_QE, (n & 1) ^ 1, 2));
          if (!ok) {
            ++it;
            break;
          }
          const int tiles = t.ntok > N * tpt ? 2 : 1;
          if (lane == 0 && rank == 0) mbar_expect_tx(BAR(C::B_QF), N * tiles * D * 2 * p.group * tpt);
          __syncwarp();
          if (lane < tiles * C::HALVES) {
            const int tl = lane / C::HALVES, hf = lane % C::HALVES, tok = t.tok + (tl * N + rank) * tpt;
            const uint32_t dst = sq + tl * C::TILE + hf * C::HALF;
            if (PAIR) tma_load_4d_pair(dst, &maps.q, hf * 64, 0, t.h, tok, even(BAR(C::B_QF)));
            else tma_load_4d(dst, &maps.q, hf * 64, 0, t.h, tok, BAR(C::B_QF));
          }
        }
        ok = __all_sync(0xffffffffu, WAIT(C::B_VE + st, ph ^ 1, 3));
        if (!ok) {
          ++it;
          break;
        }
        if (lane == 0) mbar_expect_tx(BAR(C::B_VF + st), C::STAGE);
        __syncwarp();
        if (mine) tma_load_4d(sv + st * C::STAGE + v_dst, &maps.v, v_col, t.h, vz, vw, BAR(C::B_VF + st));
        v_issued = it + 1;
      }
      if (!ok) break;
    }
    // Every copy issued lands before the block leaves.  (An odd block sees those of
    // K and Q by their use; a wait that gave up is two seconds past them.)
    if (lane == 0) {
      const int kbar = rank == 0 ? C::B_KF : C::B_KE;
      for (uint32_t i = it > ST ? it - ST : 0; i < it; ++i) mbar_drain(BAR(kbar + i % ST), (i / ST) & 1);
      for (uint32_t i = v_issued > ST ? v_issued - ST : 0; i < v_issued; ++i)
        mbar_drain(BAR(C::B_VF + i % ST), (i / ST) & 1);
      if (n) mbar_drain(BAR(rank == 0 ? C::B_QF : C::B_QE), (n - 1) & 1);
    }
  } else if (warp == 9) {
    // ----------------------------------------------------------- MMA issuer --
    if (lane == 0 && rank == 0) {
      const uint32_t ID_QK = instr_desc<T>(N * kRows, kKeys, false) | (p.negate ? 1u << 13 : 0u);   // bit 13: -A
      constexpr uint32_t ID_PV = instr_desc<T>(N * kRows, D, true);
      auto qk = [&](int t, int st) {     // S_t = Q_t K^T
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          mma_ss<PAIR>(tmem + 256 + 128 * t, smem_desc(sq + t * C::TILE + (kk >> 2) * C::HALF + (kk & 3) * 32, 16),
                       smem_desc(sk + st * C::STAGE + (kk >> 2) * C::KHALF + (kk & 3) * 32, 16), ID_QK, kk != 0);
        }
        mma_commit<PAIR>(BAR(C::B_SF + t));
      };
      auto pv = [&](int t, int st, bool acc) {   // O_t (+)= P_t V
#pragma unroll
        for (int kk = 0; kk < kKeys / 16; ++kk)
          mma_ts<PAIR>(tmem + 128 * t, tmem + 256 + 128 * t + kk * 8, smem_desc(sv + st * C::STAGE + kk * 2048, C::HALF),
                       ID_PV, (acc || kk != 0) ? 1u : 0u);
      };
      uint32_t it = 0, n = 0, seen[2] = {0, 0};
      uint32_t guarded = 0;              // parity of each place's guarded steps
      bool ok = NEXT_TASK(0);
      int a = 0, e = -1, end[2] = {0, 0}, edge = 0;
      if (ok) {
        const Task& t = TASK(0);
        a = t.a, e = t.e, end[0] = t.end[0], end[1] = t.end[1], edge = t.edge;
        mbar_arrive(BAR(C::B_TE));
      }
      bool more = e >= 0;
      int j = a;
      if (ok && more) {
        ok = WAIT(C::B_QF, 0, 4) && WAIT(C::B_KF, 0, 5);
        if (ok) {
          fence_after();
          for (int t = 0; t < 2; ++t)
            if (j < end[t]) qk(t, 0);
          mma_commit<PAIR>(BAR(C::B_KE));
          if (j + 1 == e) mma_commit<PAIR>(BAR(C::B_QE));
        }
      }
      while (more && ok) {
        // the step after this one
        int na = a, ne = e, nj = j + 1, nend[2] = {end[0], end[1]}, nedge = edge;
        const bool turn = nj == e;       // it begins another piece
        if (turn) {
          ++n;
          ok = NEXT_TASK(n);
          if (!ok) break;
          const Task& t = TASK(n);
          na = t.a, ne = t.e, nend[0] = t.end[0], nend[1] = t.end[1], nedge = t.edge;
          mbar_arrive(BAR(C::B_TE + n % kPieces));
          more = ne >= 0;
          nj = na;
        }
        const int st = it % ST, nst = (it + 1) % ST;
        bool careful = false;
        if (PAIR) {                      // both guards report every step: V's halves complete on their own blocks' barriers
          if (!WAIT(C::B_VG + st, (it / ST) & 1, 15)) break;
          if (j >= edge) {
            fence_acquire_cluster();
            careful = vflag[st * N] | vflag[st * N + N - 1];
          }
        } else if (j < edge) {
          if (!WAIT(C::B_VF + st, (it / ST) & 1, 6)) break;
        } else {
          if (!WAIT(C::B_VG + st, (guarded >> st) & 1, 15)) break;
          guarded ^= 1u << st;
          careful = vflag[st];
        }
        bool waited = false;
        for (int t = 0; t < 2 && ok; ++t) {
          if (j < end[t]) {
            ok = WAIT(C::B_PF + t, seen[t] & 1, 7 + t);
            if (!ok) break;
            ++seen[t];
            fence_after();
            if (!careful) pv(t, st, j > a);
            if (j + 1 == end[t]) mma_commit<PAIR>(BAR(C::B_OF + t));
          }
          if (t == 1) mma_commit<PAIR>(BAR(C::B_VE + st));
          if (more && nj < nend[t]) {
            if (!waited) {
              ok = (!turn || WAIT(C::B_QF, n & 1, 9)) && WAIT(C::B_KF + nst, ((it + 1) / ST) & 1, 10);
              if (!ok) break;
              fence_after();
              waited = true;
            }
            qk(t, nst);
          }
        }
        if (!ok) break;
        if (more) {
          mma_commit<PAIR>(BAR(C::B_KE + nst));
          if (nj + 1 == ne) mma_commit<PAIR>(BAR(C::B_QE));
        }
        a = na, e = ne, j = nj, end[0] = nend[0], end[1] = nend[1], edge = nedge;
        ++it;
      }
      // Every MMA issued completes before tensor memory is freed.
      mma_commit<PAIR>(BAR(C::B_END));
      mbar_drain(BAR(C::B_END), 0);
    }
  } else if (warp == 10) {
    // ---------------------------------------------------------- guard of V --
    uint32_t it = 0;
    for (uint32_t n = 0;; ++n) {
      if (!__all_sync(0xffffffffu, NEXT_TASK(n))) break;
      const Task t = TASK(n);
      __syncwarp();
      if (lane == 0) mbar_arrive(BAR(C::B_TE + n % kPieces));
      if (t.e < 0) break;
      const int some = task_visible(p, t, 0), most = task_visible(p, t, t.ntok - 1);   // seen by every row, by any
      bool ok = true;
      for (int j = t.a; j < t.e; ++j, ++it) {
        const int st = it % ST;
        ok = __all_sync(0xffffffffu, WAIT(C::B_VF + st, (it / ST) & 1, 11));
        if (!ok) break;
        int bad = 0;
        if (j >= t.edge) {
          // Rows lo.. are searched (a few more below them do no harm), rows hi.. zeroed.
          // Eight rows at a time, all loads before their use: at one load at a time
          // this took four steps' time.
          const int lo = max(0, some - j * kKeys), hi = min(kKeys, max(0, most - j * kKeys));
          constexpr int CH = D / N / 8, STEP = 32 / CH;      // 16-byte vectors of a row here; rows of one load of the warp
          const int col = lane % CH, row0 = lane / CH;
          unsigned char* v = smem + C::V0 + st * C::STAGE + (col >> 3) * C::HALF;
          uint32_t top[4] = {0, 0, 0, 0};
          for (int r8 = lo & ~7; r8 < kKeys; r8 += 8) {
            uint4 y[8 / STEP];
#pragma unroll
            for (int k = 0; k < 8 / STEP; ++k) {
              const int r = k * STEP + row0;                 // row & 7
              uint4* x = reinterpret_cast<uint4*>(v + (r8 + r) * 128 + (((col & 7) ^ r) << 4));
              if (r8 + r < hi) {
                y[k] = *x;
              } else {
                y[k] = make_uint4(0, 0, 0, 0);
                *x = y[k];
              }
            }
#pragma unroll
            for (int k = 0; k < 8 / STEP; ++k) {
              top[0] = absmax2(top[0], y[k].x);
              top[1] = absmax2(top[1], y[k].y);
              top[2] = absmax2(top[2], y[k].z);
              top[3] = absmax2(top[3], y[k].w);
            }
          }
          bad = absmax2_fold(absmax2(absmax2(top[0], top[1]), absmax2(top[2], top[3]))) >= Bits16<T>::kInf;
          fence_async_smem();
          bad = __any_sync(0xffffffffu, bad);
        } else if (!PAIR) {
          continue;
        }
        if (PAIR) {
          // to both blocks: lane r tells block r
          if (lane < N) {
            const uint32_t bar = map_to_rank(BAR(C::B_VG + st), lane);
            if (j >= t.edge) {
              st_cluster(map_to_rank(smem_u32(const_cast<int*>(vflag + st * N)) + 4 * rank, lane), bad);
              mbar_arrive_cluster<true>(bar);
            } else {
              mbar_arrive_cluster<false>(bar);
            }
          }
          __syncwarp();
        } else if (lane == 0) {
          vflag[st] = bad;
          mbar_arrive(BAR(C::B_VG + st));
        }
      }
      if (!ok) break;
    }
  } else {
    // -------------------------------------------------------------- softmax --
    const int t = warp >> 2;                       // tile of this warpgroup
    const int row = (warp & 3) * 32 + lane;        // TMEM lane
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + 256 + t * 128 + lane_off;
    const uint32_t tO = tmem + t * 128 + lane_off;
    const float c = p.scale_log2;
    const int row_tok = row / p.group;             // of this row, in its tile
    const int ti = t * N + rank;                   // the tile in its item
    const uint32_t pf = even(BAR(C::B_PF + t));
    uint32_t it = 0, tiles = 0, outs = 0, guarded = 0;
    for (uint32_t n = 0;; ++n) {
      if (!__all_sync(0xffffffffu, NEXT_TASK(n))) break;
      const Task& task = TASK(n);
      if (task.e < 0) break;
      const int a = task.a, e = task.e, end = task.end[t], first = task.edge;
      const int k_tok = ti * tpt + row_tok;        // the row's token in the item
      const int limit = task_visible(p, task, min(k_tok, task.ntok - 1));
      float m = kNoMax;                            // reference of the weights: lags behind the maximum of s * c
      float l = 0.f;                               // running sum
      bool ok = true;
      for (int j = a; j < e; ++j, ++it) {
        if (j >= first) guarded ^= 1u << (it % ST);
        if (j >= end) continue;
        ok = __all_sync(0xffffffffu, WAIT(C::B_SF + t, tiles & 1, 12));
        if (!ok) break;
        ++tiles;
        fence_after();
        float x[128];
        uint32_t* xu = reinterpret_cast<uint32_t*>(x);
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld32(tS + q * 32, xu + q * 32);
        tmem_wait_ld();
        const bool edge = j >= first;
        const int lim = limit - j * kKeys;
        if (edge) {
          // a warp's rows share most of the edge: 32 keys that all of them see are left alone
          const int least = __reduce_min_sync(0xffffffffu, lim);
#pragma unroll
          for (int q = 0; q < 128; q += 32)
            if (least < q + 32) {
#pragma unroll
              for (int i = q; i < q + 32; ++i)
                if (i >= lim) x[i] = -INFINITY;
            }
        }
        float mq[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
        for (int i = 4; i < 124; i += 8)
#pragma unroll
          for (int q = 0; q < 4; ++q) mq[q] = max3f(mq[q], x[i + 2 * q], x[i + 2 * q + 1]);
        mq[0] = max3f(mq[0], x[124], x[125]);
        mq[1] = max3f(mq[1], x[126], x[127]);
        const float mt = max3f(mq[0], mq[1], fmaxf(mq[2], mq[3])) * c;
        const bool need = mt > m + (Weight<T>::kUp + Weight<T>::kLag);
        const bool any_need = __any_sync(0xffffffffu, need);
        const float m_new = need ? mt - Weight<T>::kUp : m;
        const float alpha = ex2(m - m_new);        // 1 where the max is kept; 0 at the first visible key
        m = m_new;
        const float2 c2 = make_float2(c, c), mn2 = make_float2(-m, -m);
        float2 ra[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
        for (int ch = 0; ch < 4; ++ch) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 32 * ch; i < 32 * ch + 32; i += 2) {
            float2 w = fma2(make_float2(x[i], x[i + 1]), c2, mn2);
            w.x = ex2(w.x);
            w.y = ex2(w.y);
            pk[(i - 32 * ch) >> 1] = pack2<T>(w.x, w.y);
            ra[(i >> 1) & 3] = add2(ra[(i >> 1) & 3], w);
          }
          tmem_st16(tS + 16 * ch, pk);
        }
        const float2 r01 = add2(ra[0], ra[1]), r23 = add2(ra[2], ra[3]);
        l = __fmaf_rn(l, alpha, (r01.x + r01.y) + (r23.x + r23.y));
        // O_t *= alpha (PV_t of the step before has completed: it was issued
        // before the QK_t that released this S).
        if (any_need && j > a) {
#pragma unroll 1
          for (int q = 0; q < D; q += 32) {
            uint32_t o[32];
            tmem_ld32(tO + q, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st32(tO + q, o);
          }
        }
        tmem_wait_st();
        if (edge) {
          const int st = it % ST;
          ok = __all_sync(0xffffffffu, WAIT(C::B_VG + st, PAIR ? (it / ST) & 1 : (~guarded >> st) & 1, 13));
          if (!ok) break;
          if (PAIR) fence_acquire_cluster();
          if (vflag[st * N] | vflag[st * N + N - 1]) {
            const uint32_t v = sv + st * C::STAGE;
            careful_pv<T, D>(tS, tO, PAIR ? map_to_rank(v, 0) : v, PAIR ? map_to_rank(v, 1) : v + C::HALF, j == a, lim);
          }
        }
        fence_before();
        __syncwarp();
        if (lane == 0) {
          if (PAIR) mbar_arrive_cluster<false>(pf);
          else mbar_arrive(pf);
        }
      }
      if (!ok) break;
      // ---- epilogue ----
      const bool has = end > a;
      if (has) {
        if (!__all_sync(0xffffffffu, WAIT(C::B_OF + t, outs & 1, 14))) break;
        ++outs;
        fence_after();
      }
      const bool valid = row_tok < tpt && k_tok < task.ntok;
      const bool whole = task.slot < 0;
      Slot<D, 2 * N * kRows>& slot = static_cast<Slot<D, 2 * N * kRows>*>(maps.partial)[max(task.slot, 0)];
      const int r2 = ti * kRows + row;
      if (!whole) slot.ml[r2] = make_float2(m, l);
      if (has) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const float2 inv2 = make_float2(inv, inv);
        const uint32_t keep = l == 0.f ? 0u : 0xffffffffu;
        const int row_head = row - row_tok * p.group;
        const long long at = valid ? (long long)(task.tok + k_tok) * p.o_ts + (long long)(task.h * p.group + row_head) * p.o_hs
                                   : -1;
        long long to[4];                 // rows that this lane stores a piece of
#pragma unroll
        for (int k = 0; k < 4; ++k) to[k] = __shfl_sync(0xffffffffu, at, 8 * k + (lane >> 2));
        unsigned char* buf = smem + C::OUT + warp * 2048;
#pragma unroll 1
        for (int q = 0; q < D; q += 32) {
          uint32_t o[32];
          tmem_ld32(tO + q, o);
          tmem_wait_ld();
          // 32 columns, repaired where one that should be a number or infinity is neither
          // (ragged prompts 208-210 us, 205 without the look, 215 with loops of their own
          // for whole items and for pieces: more code to fetch)
          float2 seen = make_float2(0.f, 0.f);   // NaN where one of them is not finite
#pragma unroll
          for (int i = 0; i < 32; i += 2)
            seen = fma2(make_float2(__uint_as_float(o[i]), __uint_as_float(o[i + 1])), make_float2(0.f, 0.f), seen);
          if (__builtin_expect(__any_sync(0xffffffffu, valid && l > 0.f && seen.x + seen.y != 0.f), 0)) {
            repair_odd<T>(Values(p, task.kfirst, task.b, task.h), tO + q, q, a * kKeys, end * kKeys, limit, valid ? l : 0.f);
            tmem_ld32(tO + q, o);
            tmem_wait_ld();
          }
          if (whole) {
            // Through shared memory, so that a warp's store covers rows of 64 bytes
            // and not single 16-byte pieces of 32 of them.
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              uint32_t w[4];
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                const int c = 8 * i + 2 * k;
                const float2 x = mul2(make_float2(__uint_as_float(o[c]), __uint_as_float(o[c + 1])), inv2);
                w[k] = pack2<T>(x.x, x.y) & keep;                       // a row that sees no key is zero
              }
              *reinterpret_cast<uint4*>(buf + lane * 64 + ((i ^ (lane >> 1) & 3) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            __syncwarp();
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int r = 8 * k + (lane >> 2), i = lane & 3;
              const uint4 w = *reinterpret_cast<const uint4*>(buf + r * 64 + ((i ^ (r >> 1) & 3) << 4));
              if (to[k] >= 0) *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + to[k] + q + i * 8) = w;
            }
            __syncwarp();
          } else if (valid) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              *reinterpret_cast<uint4*>(slot.o[q / 4 + i][r2]) =
                  make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(BAR(C::B_TE + n % kPieces));
    }
  }

  fence_before();
  if (PAIR) cluster_sync(); else __syncthreads();
  fence_after();
  if (warp == 9) tmem_free_512<PAIR>(tmem);
#undef BAR
#undef WAIT
#undef NEXT_TASK
#undef TASK
}

// Joins what the tile kernel (items of TR rows) and the one for few rows (items of
// FR) left, in one launch.
template <typename T, int D, int TR, int FR>
__global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(const Params p, const ToJoin tiles, const ToJoin few) {
  __shared__ float shared[kJoinWarps][10][32];
  wait_for_primary();
  launch_dependents();
  constexpr int TY = join_y(D, TR, 1), FY = join_y(D, 32, 2);
  const int i = blockIdx.x, tile_blocks = tiles.blocks * TY;
  if (i < tile_blocks) join_item<T, D, TR, kRows, 1>(p, tiles, i / TY, i % TY, shared);
  else join_item<T, D, 32, FR, 2>(p, few, (i - tile_blocks) / FY, (i - tile_blocks) % FY, shared);
}
template <typename T, int D, int TR, int FR>
static void launch_join(const Params& p, const ToJoin& tiles, const ToJoin& few, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles.blocks * join_y(D, TR, 1) + few.blocks * join_y(D, 32, 2)));
  cfg.blockDim = dim3(32 * kJoinWarps);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, join_kernel<T, D, TR, FR>, p, tiles, few);
}

// ------------------------------------------------------------------- host --
static int64_t begun_bytes(int blocks) { return ((int64_t)blocks * (int64_t)sizeof(Begun) + 15) / 16 * 16; }
static int64_t tile_workspace(int head_dim) {
  const int n = sm_count();
  return begun_bytes(n) +
         2 * (int64_t)n * (int64_t)(head_dim == 64 ? sizeof(Slot<64, 2 * kRows>) : sizeof(Slot<128, 2 * kRows>));
}
static bool tiles_split(int64_t max_keys) { return max_keys > kWhole * kKeys; }
static int64_t workspace_bytes_for(int64_t max_keys, int head_dim) {
  return tiles_split(max_keys) || few_splits(max_keys) ? tile_workspace(head_dim) + few_workspace(head_dim) : 0;
}
static int64_t max_keys(const Params& p) { return p.table ? (int64_t)p.width * p.page : p.tokens; }
// The most K and V that a call can read, whatever the lengths are.
static int64_t kv_bytes(const Params& p) {
  int64_t keys = p.tokens;
  if (p.table) {
    const int64_t held = (int64_t)p.num_blocks * p.page, named = p.batch * max_keys(p);
    keys = held < named ? held : named;
  }
  return keys * p.kv_heads * p.head_dim * 4;
}

static int check(const char* what, Params& p, int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads,
                 int64_t head_dim, float scale, int dtype) {
  JO_REQUIRE(dtype == JO_DTYPE_BF16 || dtype == JO_DTYPE_F16, JO_ERR_DTYPE, "%s: only bf16 and fp16 are supported", what);
  JO_REQUIRE(head_dim == 64 || head_dim == 128, JO_ERR_INVALID, "%s: head_dim must be 64 or 128 (got %lld)", what,
             (long long)head_dim);
  JO_REQUIRE(tokens >= 0 && batch >= 0 && heads >= 0 && kv_heads >= 0 && tokens < (1LL << 30) && batch < (1LL << 30) &&
                 heads < 65536,
             JO_ERR_INVALID, "%s: invalid shape", what);
  JO_REQUIRE(heads == 0 || (kv_heads > 0 && heads % kv_heads == 0 && heads / kv_heads <= kRows), JO_ERR_INVALID,
             "%s: heads (%lld) must be a multiple of kv_heads (%lld), at most 128 times it", what, (long long)heads,
             (long long)kv_heads);
  // the stride of a dimension of one element is never used
  if (tokens <= 1) p.q_ts = p.o_ts = 0;
  if (tokens <= 1 && !p.table) p.k_ts = p.v_ts = 0;
  if (heads <= 1) p.q_hs = p.o_hs = 0;
  if (kv_heads <= 1) p.k_hs = p.v_hs = 0;
  if (p.num_blocks <= 1) p.k_bs = p.v_bs = 0;
  const int64_t s[10] = {p.q_ts, p.q_hs, p.k_bs, p.k_ts, p.k_hs, p.v_bs, p.v_ts, p.v_hs, p.o_ts, p.o_hs};
  for (int i = 0; i < 10; ++i)
    JO_REQUIRE(s[i] >= 0 && s[i] % 8 == 0, JO_ERR_ALIGN, "%s: strides must be non-negative multiples of 8 elements", what);
  JO_REQUIRE(aligned16(p.q) && aligned16(p.k) && aligned16(p.v) && aligned16(p.out), JO_ERR_ALIGN,
             "%s: tensors must be 16-byte aligned", what);
  JO_REQUIRE(isfinite(scale), JO_ERR_INVALID, "%s: scale must be finite", what);
  p.tokens = (int)tokens;
  p.batch = (int)batch;
  p.heads = (int)heads;
  p.kv_heads = (int)kv_heads;
  p.group = kv_heads > 0 ? (int)(heads / kv_heads) : 1;
  p.head_dim = (int)head_dim;
  // a masked score is -infinity and must stay so after the scaling, at scale 0 too
  p.scale_log2 = fmaxf(fabsf(scale) * 1.4426950408889634f, 1e-30f);
  p.negate = scale < 0.f;
  return JO_OK;
}

template <typename T, int D, bool PAIR>
static int launch_tiles(const char* what, const Params& p, void* workspace, ToJoin* join, cudaStream_t stream) {
  constexpr bool bf16 = IsBf16<T>::v;
  Maps maps;
  maps.tpt = kRows / p.group;
  constexpr int N = PAIR ? 2 : 1;
  const int units = sm_count() / N;
  const int64_t qd[4] = {D, p.group, p.kv_heads, p.tokens}, qs[3] = {p.q_hs, p.q_hs * p.group, p.q_ts};
  const int qb[4] = {64, p.group, 1, maps.tpt};
  if (!make_map_4d(&maps.q, bf16, p.q, qd, qs, qb) || !kv_maps(p, bf16, kKeys / N, &maps.k, &maps.v, &maps.box)) {
    set_error("%s: cuTensorMapEncodeTiled failed", what);
    return JO_ERR_CUDA;
  }
  const bool split = tiles_split(max_keys(p));
  maps.begun = split ? static_cast<Begun*>(workspace) : nullptr;
  maps.partial = static_cast<char*>(workspace) + begun_bytes(sm_count());
  static bool attr[kMaxDevices] = {};
  const int dev = device_slot();
  if (!attr[dev]) {
    if (cudaFuncSetAttribute(tile_kernel<T, D, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D, PAIR>::BYTES) != cudaSuccess)
      return check_launch(what);
    attr[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(units * N));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Cfg<D, PAIR>::BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = 2;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = PAIR ? 2 : 1;
  cudaLaunchKernelEx(&cfg, tile_kernel<T, D, PAIR>, maps, p);
  *join = ToJoin{maps.partial, maps.begun, split ? units : 0, maps.tpt};
  return check_launch(what);
}

// Which kernels a call takes.
struct Plan {
  bool few, tiles, pair;
};

template <typename T, int D>
static int launch_type(const char* what, Params& p, const Plan& plan, int64_t rows, int dtype, void* workspace,
                       cudaStream_t s) {
  ToJoin tiles{nullptr, nullptr, 0, 1}, few{nullptr, nullptr, 0, 1};
  FewShape shape{1};
  p.min_rows = plan.few && plan.tiles ? kFewRows + 1 : 1;
  p.max_rows = INT32_MAX;
  if (plan.tiles) {
    const int st = D == 128 && plan.pair ? launch_tiles<T, D, D == 128>(what, p, workspace, &tiles, s)
                                         : launch_tiles<T, D, false>(what, p, workspace, &tiles, s);
    if (st != JO_OK) return st;
  }
  if (plan.few) {
    // Beside the tile kernel it has requests and a workspace of its own: its blocks
    // begin as the other's end.
    Params q = p;
    q.min_rows = 1;
    if (plan.tiles) q.max_rows = kFewRows;
    const int st = launch_few(what, q, rows, dtype, static_cast<char*>(workspace) + tile_workspace(D), plan.tiles, &few,
                              &shape, s);
    if (st != JO_OK) return st;
  }
  if (tiles.blocks + few.blocks > 0) {
    if (shape.rows16 == 1) {
      if (D == 128 && plan.pair) launch_join<T, D, 4 * kRows, 16>(p, tiles, few, s);
      else launch_join<T, D, 2 * kRows, 16>(p, tiles, few, s);
    } else {
      if (D == 128 && plan.pair) launch_join<T, D, 4 * kRows, 32>(p, tiles, few, s);
      else launch_join<T, D, 2 * kRows, 32>(p, tiles, few, s);
    }
  }
  return check_launch(what);
}

static int launch(const char* what, Params& p, int64_t max_query_len, int dtype, void* workspace,
                  int64_t workspace_bytes, void* stream) {
  if (p.tokens == 0 || p.batch == 0 || p.heads == 0) return JO_OK;
  JO_REQUIRE(p.q && p.out && p.starts, JO_ERR_INVALID, "%s: null tensor pointer", what);
  int st = require_sm100();
  if (st != JO_OK) return st;
  const int64_t need = workspace_bytes_for(max_keys(p), p.head_dim);
  JO_REQUIRE(need == 0 || (workspace && aligned16(workspace) && workspace_bytes >= need), JO_ERR_INVALID,
             "%s: a 16-byte aligned workspace of %lld bytes is needed (got %lld)", what, (long long)need,
             (long long)workspace_bytes);
  // A request of few rows is bound by reading its keys and is served by its own
  // kernel.  Where the longest request is one, that kernel takes them all (in
  // runs of rows, should one be longer than announced); where a batch may hold
  // both kinds, each kernel takes its own.  (One request: the tile kernel, if it
  // can have more than few rows.)
  const int64_t longest = max_query_len < p.tokens ? (max_query_len > 1 ? max_query_len : 1) : p.tokens;
  const int64_t mean = (p.tokens + p.batch - 1) / p.batch;
  const bool only_few = p.table && p.group <= kFewRows && longest * p.group <= kFewRows;
  Plan plan;
  plan.few = only_few || (p.table && p.group <= kFewRows && p.batch > 1);
  plan.tiles = !only_few;
  plan.pair = (longest < mean ? longest : mean) * p.group >= kPairRows && kv_bytes(p) >= kPairBytes;
  const int64_t few_rows = only_few ? longest * p.group : kFewRows;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == JO_DTYPE_BF16)
    return p.head_dim == 64 ? launch_type<__nv_bfloat16, 64>(what, p, plan, few_rows, dtype, workspace, s)
                            : launch_type<__nv_bfloat16, 128>(what, p, plan, few_rows, dtype, workspace, s);
  return p.head_dim == 64 ? launch_type<__half, 64>(what, p, plan, few_rows, dtype, workspace, s)
                          : launch_type<__half, 128>(what, p, plan, few_rows, dtype, workspace, s);
}

}  // namespace vattn
}  // namespace jo

extern "C" {

int jo_paged_attention(const void* q, const void* key_cache, const void* value_cache, const int32_t* block_tables,
                       const int32_t* query_starts, const int32_t* kv_lens, void* out, int64_t tokens, int64_t batch,
                       int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t num_blocks, int64_t page_size,
                       int64_t table_width, int64_t table_stride, const int64_t* row_strides,
                       const int64_t* cache_strides, int causal, float scale, int64_t max_query_len, int dtype,
                       void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace jo;
  const char* what = "paged_attention";
  JO_REQUIRE(row_strides && cache_strides, JO_ERR_INVALID, "%s: null strides", what);
  const int64_t *r = row_strides, *c = cache_strides;
  JO_REQUIRE(page_size >= 16 && page_size % 16 == 0 && page_size < (1LL << 30), JO_ERR_INVALID,
             "%s: page_size must be a multiple of 16 (got %lld)", what, (long long)page_size);
  JO_REQUIRE(num_blocks >= 0 && num_blocks < (1LL << 31) && table_width >= 0 && table_width < (1LL << 31) &&
                 table_stride >= 0 && table_width * page_size <= (1LL << 30),
             JO_ERR_INVALID, "%s: invalid cache or block table shape", what);
  // (a table without columns is never read, but says that there is one)
  vattn::Params p{q, key_cache, value_cache, out, query_starts, kv_lens, table_width > 0 ? block_tables : query_starts,
                  r[0], r[1], c[0], c[1], c[2], c[3], c[4], c[5], r[2], r[3], table_stride};
  p.num_blocks = (int)num_blocks;
  p.page = (int)page_size;
  p.width = (int)table_width;
  p.causal = causal != 0;
  int st = vattn::check(what, p, tokens, batch, heads, kv_heads, head_dim, scale, dtype);
  if (st != JO_OK) return st;
  JO_REQUIRE(tokens == 0 || batch == 0 || (kv_lens && (block_tables || table_width == 0) &&
                                            (num_blocks == 0 || (key_cache && value_cache))),
             JO_ERR_INVALID, "%s: null tensor pointer", what);
  return vattn::launch(what, p, max_query_len, dtype, workspace, workspace_bytes, stream);
}

int jo_prompt_attention(const void* q, const void* k, const void* v, const int32_t* seq_starts, void* out,
                        int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                        const int64_t* row_strides, const int64_t* kv_strides, int causal, float scale, int dtype,
                        void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace jo;
  const char* what = "prompt_attention";
  JO_REQUIRE(row_strides && kv_strides, JO_ERR_INVALID, "%s: null strides", what);
  const int64_t *r = row_strides, *c = kv_strides;
  vattn::Params p{q, k, v, out, seq_starts, nullptr, nullptr, r[0], r[1], 0, c[0], c[1], 0, c[2], c[3], r[2], r[3], 0};
  p.num_blocks = 0;
  p.page = 1;
  p.width = 0;
  p.causal = causal != 0;
  int st = vattn::check(what, p, tokens, batch, heads, kv_heads, head_dim, scale, dtype);
  if (st != JO_OK) return st;
  JO_REQUIRE(tokens == 0 || batch == 0 || (k && v), JO_ERR_INVALID, "%s: null tensor pointer", what);
  return vattn::launch(what, p, tokens, dtype, workspace, workspace_bytes, stream);
}

int jo_varlen_attention_workspace(int64_t max_keys, int64_t head_dim, int64_t* bytes) {
  using namespace jo;
  JO_REQUIRE(bytes, JO_ERR_INVALID, "varlen_attention_workspace: null pointer");
  JO_REQUIRE(head_dim == 64 || head_dim == 128, JO_ERR_INVALID,
             "varlen_attention_workspace: head_dim must be 64 or 128 (got %lld)", (long long)head_dim);
  *bytes = vattn::workspace_bytes_for(max_keys, (int)head_dim);
  return JO_OK;
}

// Fault code of the kernels' bounded waits (0 = none); reset != 0 clears it.
// One sticky value per device, shared by every launch.  Synchronous.
int jo_varlen_attention_last_fault(int reset) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, jo::vattn::g_fault, sizeof(int)) != cudaSuccess) {
    cudaGetLastError();
    return JO_ERR_CUDA;
  }
  if (reset) {
    int z = 0;
    cudaMemcpyToSymbol(jo::vattn::g_fault, &z, sizeof(int));
  }
  const int w = jo::vattn::few_last_fault(reset);
  return v != 0 ? v : w;
}

}  // extern "C"
