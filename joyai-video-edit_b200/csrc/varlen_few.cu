// Attention over a paged cache for requests of few rows (single tokens, or a
// few, times the heads of a group): up to 32 rows of one key head at a time.
//
// Bound by reading K and V once: 4 * head_dim bytes a key for at most 32 rows'
// worth of arithmetic.  So the organisation is the one that keeps the most bytes
// in flight with the least work per byte: two blocks on every SM, each with 96 KB
// of K and V steps (64 keys) on the way through TMA, looked after by one warp,
// and four warps on mma.sync (m16n8k16: its 16 rows fit a group, where the 128 of
// a tcgen05 tile would be mostly empty).  Of a step's scores each warp has 16
// keys, of its output a quarter of the columns; the weights change hands in
// shared memory, with two barriers a step.  The steps of all items are shared out
// evenly over the blocks (varlen_attention.cuh).
//
// Measured, the join included: one token over 131071 cached ones (32 heads over 8
// of 128, 537 MB) 99-102 us, 5.3-5.4 TB/s; 64 single tokens over 54480 (224 MB) 49-50
// us; one over 300 (14 heads over 2 of 64) 8.1 us, nearly all of it latency.
#include "varlen_attention.cuh"

namespace jo {
namespace vattn {
namespace few {

constexpr int kKeys = 64;                // keys of a step
constexpr int kWarps = 4;                // warps that compute
constexpr int kThreads = 32 * (kWarps + 1);
// Steps that an item's beginning and end cost; steps of the shortest piece; items
// that are never cut (300 tokens, five steps: 8.1 us, in two pieces and a join 10.1;
// 440, seven steps: 10.5 and 9.6, with the join's launch in both, since the table has
// room for more; 4000: 11.3 us, in pieces of four at least 13.6).
constexpr int kLead = 2, kMin = 2, kWhole = 7;
constexpr int kBlocksPerSm = 2;

using Steps = Work<kKeys, kLead, kMin, kWhole>;
using Range = Steps::Range;
using Piece = Steps::Piece;
using Walk = Steps::Walk;

__device__ int g_fault = 0;

template <int D, int MT> struct Cfg {
  static constexpr int R = 16 * MT;                          // rows of an item
  static constexpr int HALVES = D / 64, HALF = kKeys * 128;  // 64 columns: 128-byte rows
  static constexpr int TILE = HALVES * HALF;                 // K or V of a step
  static constexpr int ST = D == 128 ? 3 : 6;                // steps in flight: 96 KB
  static constexpr int Q0 = ST * 2 * TILE;                   // Q: R rows, 16-byte pieces turned as the swizzle does
  static constexpr int P0 = Q0 + R * D * 2;                  // weights: R rows of 64 keys, likewise; rounded, then the rest
  static constexpr int P_BYTES = R * kKeys * 2;
  static constexpr int BARS = P0 + 2 * P_BYTES;
  static constexpr int NEAR = BARS + 128;
  static constexpr int BYTES = NEAR + (int)sizeof(Steps::Near);
  static_assert(2 * ST * 8 + 4 <= 128, "");
  static_assert(kWarps * R * 4 <= P_BYTES, "");
  static_assert(BYTES + 1024 <= 228 * 1024 / kBlocksPerSm, "");
};

struct Maps {
  CUtensorMap k, v;
  int box;                               // keys of one copy
  int tpi;                               // tokens of an item
  int beside;                            // runs beside the kernel before it, and needs nothing of it
  void* partial;
  Begun* begun;
};

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <typename T> __device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The barrier of the computing warps, and the one that tells whether any thread's flag is set.
__device__ __forceinline__ void team_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory"); }

__device__ __forceinline__ bool team_any(bool flag) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 q, %1, 0;\n bar.red.or.pred p, 1, %2, q;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(r)
      : "r"((uint32_t)flag), "n"(32 * kWarps)
      : "memory");
  return r != 0;
}

template <typename T, int D, int MT>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) few_kernel(const __grid_constant__ Maps maps, const Params p) {
  using C = Cfg<D, MT>;
  constexpr int ST = C::ST, R = C::R;
  extern __shared__ __align__(1024) unsigned char smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::BARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 2 * ST);
  Steps::Near& near = *reinterpret_cast<Steps::Near*>(smem + C::NEAR);
  const uint32_t bar0 = smem_u32(bars), ring = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#define FULL(s) (bar0 + 8u * (uint32_t)(s))
#define EMPTY(s) (bar0 + 8u * (uint32_t)(ST + (s)))

  if (!maps.beside) wait_for_primary();
  const Request early = (int)threadIdx.x < p.batch ? request(p, threadIdx.x) : Request{0, 0, 0};
  launch_dependents();
  if (threadIdx.x == 0) {
    tma_prefetch_map(&maps.k);
    tma_prefetch_map(&maps.v);
    for (int s = 0; s < ST; ++s) {
      mbar_init(FULL(s), 1);
      mbar_init(EMPTY(s), kWarps);
    }
    // The swizzle goes by address bits: without static shared memory the
    // dynamic part begins on a 1024-byte boundary.
    *abort_flag = (ring & 1023u) != 0;
    if (*abort_flag) atomicCAS(&g_fault, 0, 100);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  Range range;
  using Scan = Steps::Scan<kThreads / 32>;
  Steps::find<kThreads / 32>(p, early, maps.tpi, blockIdx.x, gridDim.x, *reinterpret_cast<Scan*>(smem), near, range);
  fence_async_smem();                    // the scan's space becomes the ring
  __syncthreads();
  const int tpi = maps.tpi;
  Walk walk(p, tpi, near, range);
  Piece s;
  bool ok = !*abort_flag;

  if (warp == kWarps) {
    // ------------------------------------------------------------- producer --
    const int boxes = kKeys / maps.box;
    const int bx = lane % boxes, part = lane / boxes;        // this lane's copy: K or V, 64 columns, keys
    const bool mine = lane < boxes * C::HALVES * 2;
    const int half = part % C::HALVES;
    const CUtensorMap* map = part < C::HALVES ? &maps.k : &maps.v;
    const uint32_t dst = part * C::HALF + bx * maps.box * 128;
    uint32_t it = 0;
    Begun begun{0, 0, 0, 0};
    while (ok && walk.next(s)) {
      if (s.a == 0 && s.e < s.steps)     // only the last piece ends inside an item
        begun = Begun{Steps::later_blocks(range, s, blockIdx.x), s.r.first + s.i * tpi, min(tpi, s.r.n - s.i * tpi), s.h};
      int z = 0, w = 0;                  // places of 16 keys each, eight steps at a time: pages are multiples of 16 keys
      for (int j = s.a; j < s.e; ++j, ++it) {
        const int st = it % ST, ahead = (j - s.a) & 7;
        if (ahead == 0) kv_place(p, s.r.first, s.r.keys, s.b, j * kKeys + lane * 16, z, w);
        const int from = (ahead * 4 + bx * (maps.box / 16)) & 31;
        const int zz = __shfl_sync(0xffffffffu, z, from), ww = __shfl_sync(0xffffffffu, w, from);
        ok = __all_sync(0xffffffffu, mbar_wait(EMPTY(st), ((it / ST) & 1) ^ 1, abort_flag, &g_fault, 101));
        if (!ok) break;
        if (lane == 0) mbar_expect_tx(FULL(st), 2 * C::TILE);
        __syncwarp();
        if (mine) tma_load_4d(ring + st * 2 * C::TILE + dst, map, half * 64, s.h, zz, ww, FULL(st));
      }
    }
    if (lane == 0) {
      if (maps.begun) maps.begun[blockIdx.x] = ok ? begun : Begun{0, 0, 0, 0};
      // every copy issued lands before the block leaves
      for (uint32_t i = it > ST ? it - ST : 0; i < it; ++i) mbar_drain(FULL(i % ST), (i / ST) & 1);
    }
  } else {
    // -------------------------------------------------------------- compute --
    constexpr int NW = D / 8 / kWarps;                       // 8-column blocks of this warp's output
    const int qr = lane >> 2, qc = (lane & 3) * 2;           // row and columns of this lane in a fragment
    const float c = p.scale_log2;
    // ldmatrix: row and 8-column block that this lane points at
    const int krow = warp * 16 + (lane >> 4) * 8 + (lane & 7), kcol = (lane >> 3) & 1;
    const int vrow = ((lane >> 3) & 1) * 8 + (lane & 7), vcol = lane >> 4;
    const int arow = lane & 15, acol = lane >> 4;
    const uint32_t qs = ring + C::Q0, ps = ring + C::P0;
    uint32_t it = 0;
    // After a wait that gave up the warps still go through all steps, without further
    // waits: they meet at barriers, which have no limit.  What they compute and store
    // from there is of no use, and the fault code is what tells; into the ring, where a
    // late copy may still land, they write nothing.
    while (walk.next(s)) {
      const int tok0 = s.i * tpi, ntok = min(tpi, s.r.n - tok0);
      const int some = visible(p, s.r, tok0), most = visible(p, s.r, tok0 + ntok - 1);
      for (int i = threadIdx.x; i < R * (D / 8); i += 32 * kWarps) {
        const int r = i / (D / 8), n = i % (D / 8), tok = r / p.group, g = r - tok * p.group;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (tok < ntok) {
          x = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + (int64_t)(s.r.first + tok0 + tok) * p.q_ts +
                                              (int64_t)(s.h * p.group + g) * p.q_hs + n * 8);
          if (p.negate) x.x ^= 0x80008000u, x.y ^= 0x80008000u, x.z ^= 0x80008000u, x.w ^= 0x80008000u;
        }
        *reinterpret_cast<uint4*>(smem + C::Q0 + r * D * 2 + ((n ^ (r & 7)) << 4)) = x;
      }
      int limit[MT][2];                                      // keys that this lane's rows see
      float o[MT][NW][4], m[MT][2], l[MT][2];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int tok = (t * 16 + e * 8 + qr) / p.group;
          limit[t][e] = tok < ntok ? visible(p, s.r, tok0 + tok) : 0;
          m[t][e] = kNoMax;
          l[t][e] = 0.f;
        }
#pragma unroll
        for (int n = 0; n < NW; ++n) o[t][n][0] = o[t][n][1] = o[t][n][2] = o[t][n][3] = 0.f;
      }
      team_sync();
      for (int j = s.a; j < s.e; ++j, ++it) {
        const int st = it % ST;
        ok = ok && __all_sync(0xffffffffu, mbar_wait(FULL(st), (it / ST) & 1, abort_flag, &g_fault, 102));
        const uint32_t ks = ring + st * 2 * C::TILE, vs = ks + C::TILE;
        const int key0 = j * kKeys + warp * 16;              // this warp's keys
        float x[MT][2][4], x2[MT][2][4];                     // even and odd products apart: half the chain
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[t][n][i] = x2[t][n][i] = 0.f;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          uint32_t b[4];
          ldsm4(ks + (k >> 2) * C::HALF + krow * 128 + ((((k & 3) * 2 + kcol) ^ (krow & 7)) << 4), b);
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            uint32_t a[4];
            ldsm4(qs + (t * 16 + arow) * D * 2 + (((k * 2 + acol) ^ (arow & 7)) << 4), a);
            mma16816<T>(k & 1 ? x2[t][0] : x[t][0], a, b[0], b[1]);
            mma16816<T>(k & 1 ? x2[t][1] : x[t][1], a, b[2], b[3]);
          }
        }
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[t][n][i] += x2[t][n][i];
        const bool edge = (j + 1) * kKeys > some;            // some row does not see every key of this step
        int bad = 0;
        if (edge && ok) {
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (key0 + n * 8 + qc + (i & 1) >= limit[t][i >> 1]) x[t][n][i] = -INFINITY;
          // a product with a weight of 0 would turn a NaN in V into NaN: in this
          // warp's columns, keys that no row sees are zeroed, others are searched
          // (some rows below the first partly visible one are looked at too)
          constexpr int STEP = 32 / NW;                      // rows of one load of the warp
          const int col = warp * NW + lane % NW, row0 = lane / NW;
          const int hi = most - j * kKeys;
          unsigned char* v = smem + st * 2 * C::TILE + C::TILE + (col >> 3) * C::HALF;
          uint32_t big = 0;
          for (int r0 = max(0, some - j * kKeys) & ~(2 * STEP - 1); r0 < kKeys; r0 += 2 * STEP) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int r = r0 + k * STEP + row0;
              uint4* y = reinterpret_cast<uint4*>(v + r * 128 + (((col ^ r) & 7) << 4));
              if (r < hi) {
                const uint4 u = *y;
                big = absmax2(absmax2(absmax2(absmax2(big, u.x), u.y), u.z), u.w);
              } else {
                *y = make_uint4(0, 0, 0, 0);
              }
            }
          }
          bad = absmax2_fold(big) >= Bits16<T>::kInf;
          fence_async_smem();                                // the next copy into this place comes after these writes
          bad = __any_sync(0xffffffffu, bad);
        }
        // m only moves when the maximum has grown by more than kLag somewhere.
        constexpr float kGrown = Weight<T>::kUp + Weight<T>::kLag;
        float top[MT][2];
        bool raise = false;
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(fmaxf(x[t][0][2 * e], x[t][0][2 * e + 1]), fmaxf(x[t][1][2 * e], x[t][1][2 * e + 1]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            top[t][e] = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)) * c;
            raise |= top[t][e] > m[t][e] + kGrown;
          }
        if (team_any(raise)) {                               // (all are past the step before: its weights' place is free)
          float* tops = reinterpret_cast<float*>(smem + C::P0);
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if ((lane & 3) == 0) tops[warp * R + t * 16 + e * 8 + qr] = top[t][e];
          team_sync();
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              float mx = kNoMax;
#pragma unroll
              for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, tops[w * R + t * 16 + e * 8 + qr]);
              const float mn = mx > m[t][e] + kGrown ? mx - Weight<T>::kUp : m[t][e], alpha = ex2(m[t][e] - mn);
              m[t][e] = mn;
              l[t][e] *= alpha;
#pragma unroll
              for (int n = 0; n < NW; ++n) {
                o[t][n][2 * e] *= alpha;
                o[t][n][2 * e + 1] *= alpha;
              }
            }
          team_sync();
        }
        // The weights, as the sum of two numbers of the tensors' type, so that the
        // product with V keeps 16 bits of them and more (fp16: of those above 2^-20 of
        // the largest; of smaller ones all multiples of 2^-35).  (Rounded once, they made the
        // result's error 1.4 times that of rounding it; this costs 0.4 us of 8 at one
        // short request and 0.5-1 % at the others.)
        float sum[MT][2];
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = t * 16 + e * 8 + qr;
            sum[t][e] = 0.f;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
              const float a = ex2(fmaf(x[t][n][2 * e], c, -m[t][e])), b = ex2(fmaf(x[t][n][2 * e + 1], c, -m[t][e]));
              sum[t][e] += a + b;
              const uint32_t hi = pack2<T>(a, b);
              const float2 h = unpack2<T>(hi);
              unsigned char* at = smem + C::P0 + r * 128 + (((warp * 2 + n) ^ (r & 7)) << 4) + qc * 2;
              *reinterpret_cast<uint32_t*>(at) = hi;
              *reinterpret_cast<uint32_t*>(at + C::P_BYTES) = pack2<T>(a - h.x, b - h.y);
            }
          }
        team_sync();
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          l[t][0] += sum[t][0];
          l[t][1] += sum[t][1];
        }
        if (!bad) {
#pragma unroll
          for (int k = 0; k < kKeys / 16; ++k) {
            uint32_t a[MT][4], rest[MT][4];
#pragma unroll
            for (int t = 0; t < MT; ++t) {
              const uint32_t at = ps + (t * 16 + arow) * 128 + (((k * 2 + acol) ^ (arow & 7)) << 4);
              ldsm4(at, a[t]);
              ldsm4(at + C::P_BYTES, rest[t]);
            }
#pragma unroll
            for (int n = 0; n < NW / 2; ++n) {
              const int col = warp * NW + 2 * n + vcol;      // 8-column block
              uint32_t b[4];
              ldsm4_t(vs + (col >> 3) * C::HALF + (k * 16 + vrow) * 128 + (((col & 7) ^ (vrow & 7)) << 4), b);
#pragma unroll
              for (int t = 0; t < MT; ++t) {
                mma16816<T>(o[t][2 * n], a[t], b[0], b[1]);
                mma16816<T>(o[t][2 * n + 1], a[t], b[2], b[3]);
                mma16816<T>(o[t][2 * n], rest[t], b[0], b[1]);
                mma16816<T>(o[t][2 * n + 1], rest[t], b[2], b[3]);
              }
            }
          }
        } else {
          // a NaN or infinity that only some rows may see: row by row on the CUDA cores
          const unsigned char* v = smem + st * 2 * C::TILE + C::TILE;
#pragma unroll 1
          for (int k = 0; k < kKeys; ++k) {
#pragma unroll
            for (int n = 0; n < NW; ++n) {
              const float2 f =
                  unpack2<T>(*reinterpret_cast<const uint32_t*>(v + swizzled(k, (warp * NW + n) * 8 + qc, C::HALF)));
#pragma unroll
              for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  if (j * kKeys + k < limit[t][e]) {
                    const int r = t * 16 + e * 8 + qr;
                    const T* at = reinterpret_cast<const T*>(smem + C::P0 + r * 128 + (((k >> 3) ^ (r & 7)) << 4) + (k & 7) * 2);
                    const float w = to_f32(at[0]) + to_f32(at[C::P_BYTES / 2]);
                    o[t][n][2 * e] = fmaf(w, f.x, o[t][n][2 * e]);
                    o[t][n][2 * e + 1] = fmaf(w, f.y, o[t][n][2 * e + 1]);
                  }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(EMPTY(st));
      }
      // ---- the rows' sums over the four warps, then the result ----
      team_sync();                                           // the weights have been read
      float* sums = reinterpret_cast<float*>(smem + C::P0);
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 1);
          l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 2);
          if ((lane & 3) == 0) sums[warp * R + t * 16 + e * 8 + qr] = l[t][e];
        }
      team_sync();
      float total[MT][2];                                    // the rows' sums of weights
      bool nan = false;                                      // in a row whose weights are numbers
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float seen = 0.f;                                  // NaN where a sum is not finite
          total[t][e] = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) total[t][e] += sums[w * R + t * 16 + e * 8 + qr];
#pragma unroll
          for (int n = 0; n < NW; ++n) seen = fmaf(o[t][n][2 * e], 0.f, fmaf(o[t][n][2 * e + 1], 0.f, seen));
          nan |= seen != seen && total[t][e] > 0.f;
        }
      const bool odd = __any_sync(0xffffffffu, nan);
      const bool whole = s.whole();
      Slot<D, 32>& slot = static_cast<Slot<D, 32>*>(maps.partial)[2 * blockIdx.x + (s.a == 0 ? 1 : 0)];
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = t * 16 + e * 8 + qr, tok = r / p.group, g = r - tok * p.group;
          const float sum = total[t][e];
          if (odd) {
            const Values values(p, s.r.first, s.b, s.h);
#pragma unroll
            for (int n = 0; n < NW; ++n) {
              const uint32_t need = (is_odd(o[t][n][2 * e], sum) ? 1u : 0u) | (is_odd(o[t][n][2 * e + 1], sum) ? 2u : 0u);
              float x[8];
              odd_values<T>(values, (warp * NW + n) * 8, need << qc, s.a * kKeys, some, min(s.e * kKeys, most), limit[t][e], x);
              o[t][n][2 * e] = with_odd(o[t][n][2 * e], x[qc], sum);
              o[t][n][2 * e + 1] = with_odd(o[t][n][2 * e + 1], x[qc + 1], sum);
            }
          }
          if (tok >= ntok) continue;
          if (whole) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            T* row = static_cast<T*>(p.out) + (int64_t)(s.r.first + tok0 + tok) * p.o_ts + (int64_t)(s.h * p.group + g) * p.o_hs +
                     warp * NW * 8 + qc;
#pragma unroll
            for (int n = 0; n < NW; ++n)
              *reinterpret_cast<uint32_t*>(row + n * 8) = pack2<T>(o[t][n][2 * e] * inv, o[t][n][2 * e + 1] * inv);
          } else {
            if (warp == 0 && (lane & 3) == 0) slot.ml[r] = make_float2(m[t][e], sum);
#pragma unroll
            for (int n = 0; n < NW; ++n) {
              const int col = (warp * NW + n) * 8 + qc;
              *reinterpret_cast<float2*>(&slot.o[col / 4][r][col % 4]) = make_float2(o[t][n][2 * e], o[t][n][2 * e + 1]);
            }
          }
        }
    }
  }
  // The kernel does not end before the ones ahead of it: one block sees to that,
  // the others make room.
  if (maps.beside && blockIdx.x == 0) wait_for_primary();
#undef FULL
#undef EMPTY
}

static int64_t begun_bytes(int blocks) { return ((int64_t)blocks * (int64_t)sizeof(Begun) + 15) / 16 * 16; }

template <typename T, int D, int MT>
static int launch(const char* what, const Params& p, void* workspace, bool beside, ToJoin* join, cudaStream_t stream) {
  using C = Cfg<D, MT>;
  Maps maps;
  if (!kv_maps(p, IsBf16<T>::v, kKeys, &maps.k, &maps.v, &maps.box)) {
    set_error("%s: cuTensorMapEncodeTiled failed", what);
    return JO_ERR_CUDA;
  }
  const int blocks = kBlocksPerSm * sm_count();
  maps.tpi = C::R / p.group;
  maps.beside = beside;
  const bool split = few_splits((int64_t)p.width * p.page);
  maps.begun = split ? static_cast<Begun*>(workspace) : nullptr;
  maps.partial = static_cast<char*>(workspace) + begun_bytes(blocks);
  static bool attr[kMaxDevices] = {};
  const int dev = device_slot();
  if (!attr[dev]) {
    if (cudaFuncSetAttribute(few_kernel<T, D, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::BYTES) != cudaSuccess)
      return check_launch(what);
    attr[dev] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, few_kernel<T, D, MT>, maps, p);
  *join = ToJoin{maps.partial, maps.begun, split ? blocks : 0, maps.tpi};
  return check_launch(what);
}

template <typename T, int D>
static int launch_rows(const char* what, const Params& p, int mt, void* workspace, bool beside, ToJoin* join,
                       cudaStream_t stream) {
  return mt == 1 ? launch<T, D, 1>(what, p, workspace, beside, join, stream)
                 : launch<T, D, 2>(what, p, workspace, beside, join, stream);
}

}  // namespace few

bool few_splits(int64_t max_keys) { return max_keys > few::kWhole * few::kKeys; }

int64_t few_workspace(int head_dim) {
  const int n = few::kBlocksPerSm * sm_count();
  return few::begun_bytes(n) + 2 * (int64_t)n * (int64_t)(head_dim == 64 ? sizeof(Slot<64, 32>) : sizeof(Slot<128, 32>));
}

int launch_few(const char* what, const Params& p, int64_t rows, int dtype, void* workspace, bool beside, ToJoin* join,
               FewShape* shape, cudaStream_t s) {
  const int mt = shape->rows16 = rows <= 16 ? 1 : 2;
  if (dtype == JO_DTYPE_BF16)
    return p.head_dim == 64 ? few::launch_rows<__nv_bfloat16, 64>(what, p, mt, workspace, beside, join, s)
                            : few::launch_rows<__nv_bfloat16, 128>(what, p, mt, workspace, beside, join, s);
  return p.head_dim == 64 ? few::launch_rows<__half, 64>(what, p, mt, workspace, beside, join, s)
                          : few::launch_rows<__half, 128>(what, p, mt, workspace, beside, join, s);
}

int few_last_fault(int reset) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, few::g_fault, sizeof(int)) != cudaSuccess) {
    cudaGetLastError();
    return JO_ERR_CUDA;
  }
  if (reset) {
    int z = 0;
    cudaMemcpyToSymbol(few::g_fault, &z, sizeof(int));
  }
  return v;
}

}  // namespace vattn
}  // namespace jo
