// Attention over a paged cache for requests of few rows (single tokens, or a
// few, times the heads of a group): up to 32 rows of one key head at a time.
//
// Bound by reading K and V once: 4 * head_dim bytes a key for at most 32 rows'
// worth of arithmetic.  So the organisation is the one that keeps the most bytes
// in flight with the least work per byte: two blocks on every SM, each with 96 KB
// of K and V steps (64 keys) on the way through TMA, looked after by one warp,
// and four warps that take 16 keys of a step each with mma.sync (m16n8k16: its 16
// rows fit a group, where the 128 of a tcgen05 tile would be mostly empty).  The
// four warps keep maxima, sums and accumulators of their own and meet only at the
// end of an item's piece, not at every step.  The steps of all items are shared
// out evenly over the blocks (varlen_attention.cuh).
#include "varlen_attention.cuh"

namespace jo {
namespace vattn {
namespace few {

constexpr int kKeys = 64;                // keys of a step
constexpr int kWarps = 4;                // warps that compute
constexpr int kThreads = 32 * (kWarps + 1);
constexpr int kLead = 3;                 // steps that an item's beginning and end cost
constexpr int kMin = 4;                  // steps of the shortest piece
constexpr int kBlocksPerSm = 2;

using Steps = Work<kKeys, kLead, kMin>;
using Range = Steps::Range;
using Piece = Steps::Piece;
using Walk = Steps::Walk;

__device__ int g_fault = 0;

template <int D, int MT> struct Cfg {
  static constexpr int R = 16 * MT;                          // rows of an item
  static constexpr int HALVES = D / 64, HALF = kKeys * 128;  // 64 columns: 128-byte rows
  static constexpr int TILE = HALVES * HALF;                 // K or V of a step
  static constexpr int ST = D == 128 ? 3 : 6;                // steps in flight: 96 KB
  // During the steps: Q, then weights of the careful product.  After them: the
  // warps' maxima and sums, then the R x D result in fp32.
  static constexpr int MERGE = ST * 2 * TILE;
  static constexpr int WEIGHTS = R * D * 2;
  static constexpr int SPACE = WEIGHTS + kWarps * R * 64 > R * D * 4 ? WEIGHTS + kWarps * R * 64 : R * D * 4;
  static constexpr int BARS = MERGE + SPACE;
  static constexpr int NEAR = BARS + 128;
  static constexpr int BYTES = NEAR + (int)sizeof(Steps::Near);
  static_assert(2 * ST * 8 + 4 <= 128, "");
  static_assert(BYTES + 1024 <= 228 * 1024 / kBlocksPerSm, "");
  static_assert(sizeof(Steps::Scan) <= (size_t)MERGE, "");
};

struct Maps {
  CUtensorMap k, v;
  int box;                               // keys of one copy
  int tpi;                               // tokens of an item
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
// The barrier of the computing warps.
__device__ __forceinline__ void team_sync() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kWarps) : "memory"); }

template <typename T, int D, int MT>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) few_kernel(const __grid_constant__ Maps maps, const Params p) {
  using C = Cfg<D, MT>;
  constexpr int ST = C::ST, R = C::R;
  extern __shared__ __align__(1024) unsigned char smem[];
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::BARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 2 * ST);
  float* merge = reinterpret_cast<float*>(smem + C::MERGE);
  Steps::Near& near = *reinterpret_cast<Steps::Near*>(smem + C::NEAR);
  const uint32_t bar0 = smem_u32(bars), ring = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#define FULL(s) (bar0 + 8u * (uint32_t)(s))
#define EMPTY(s) (bar0 + 8u * (uint32_t)(ST + (s)))

  launch_dependents();
  if (threadIdx.x == 0) {
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
  Steps::find<kThreads>(p, maps.tpi, blockIdx.x, gridDim.x, *reinterpret_cast<Steps::Scan*>(smem), near, range);
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
        if (ahead == 0) kv_place(p, s.r, s.b, j * kKeys + lane * 16, z, w);
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
    const int qr = lane >> 2, qc = (lane & 3) * 2;           // row and columns of this lane in a fragment
    const float c = p.scale_log2;
    // ldmatrix: row and 8-column block that this lane points at
    const int krow = warp * 16 + (lane >> 4) * 8 + (lane & 7), kcol = (lane >> 3) & 1;
    const int vrow = warp * 16 + ((lane >> 3) & 1) * 8 + (lane & 7), vcol = lane >> 4;
    const int qrow = lane & 15, qcol = lane >> 4;
    const uint32_t qs = ring + C::MERGE;
    uint32_t it = 0;
    // After a wait that gave up the warps skip the steps but still walk the pieces:
    // they meet at the barriers below, which have no limit.
    while (walk.next(s)) {
      const int tok0 = s.i * tpi, ntok = min(tpi, s.r.n - tok0);
      const int some = visible(p, s.r, tok0), most = visible(p, s.r, tok0 + ntok - 1);
      // Q, in 16-byte pieces turned by the row as the swizzle does
      for (int i = threadIdx.x; i < R * (D / 8); i += 32 * kWarps) {
        const int r = i / (D / 8), n = i % (D / 8), tok = r / p.group, g = r - tok * p.group;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (tok < ntok) {
          x = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + (int64_t)(s.r.first + tok0 + tok) * p.q_ts +
                                              (int64_t)(s.h * p.group + g) * p.q_hs + n * 8);
          if (p.negate) x.x ^= 0x80008000u, x.y ^= 0x80008000u, x.z ^= 0x80008000u, x.w ^= 0x80008000u;
        }
        *reinterpret_cast<uint4*>(smem + C::MERGE + r * D * 2 + ((n ^ (r & 7)) << 4)) = x;
      }
      int limit[MT][2];                                      // keys that this lane's rows see
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int tok = (t * 16 + e * 8 + qr) / p.group;
          limit[t][e] = tok < ntok ? visible(p, s.r, tok0 + tok) : 0;
        }
      float o[MT][D / 8][4], m[MT][2], l[MT][2];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        m[t][0] = m[t][1] = kNoMax;
        l[t][0] = l[t][1] = 0.f;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) o[t][n][0] = o[t][n][1] = o[t][n][2] = o[t][n][3] = 0.f;
      }
      team_sync();
      for (int j = s.a; j < s.e && ok; ++j, ++it) {
        const int st = it % ST;
        ok = __all_sync(0xffffffffu, mbar_wait(FULL(st), (it / ST) & 1, abort_flag, &g_fault, 102));
        if (!ok) break;
        const uint32_t ks = ring + st * 2 * C::TILE, vs = ks + C::TILE;
        const int key0 = j * kKeys + warp * 16;              // this warp's keys
        float x[MT][2][4];
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int n = 0; n < 2; ++n) x[t][n][0] = x[t][n][1] = x[t][n][2] = x[t][n][3] = 0.f;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          uint32_t b[4];
          ldsm4(ks + (k >> 2) * C::HALF + krow * 128 + ((((k & 3) * 2 + kcol) ^ (krow & 7)) << 4), b);
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            uint32_t a[4];
            ldsm4(qs + (t * 16 + qrow) * D * 2 + (((k * 2 + qcol) ^ (qrow & 7)) << 4), a);
            mma16816<T>(x[t][0], a, b[0], b[1]);
            mma16816<T>(x[t][1], a, b[2], b[3]);
          }
        }
        int bad = 0;
        if (key0 + 16 > some) {                              // some row does not see every key
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (key0 + n * 8 + qc + (i & 1) >= limit[t][i >> 1]) x[t][n][i] = -INFINITY;
          // a product with a weight of 0 would turn a NaN in V into NaN: rows
          // that no query row sees are zeroed, others are searched
          unsigned char* v = smem + st * 2 * C::TILE + C::TILE;
          constexpr int CH = D / 8;
          for (int i = max(0, some - key0) * CH + lane; i < 16 * CH; i += 32) {
            const int row = i / CH;
            uint4* y = reinterpret_cast<uint4*>(v + swizzled(warp * 16 + row, (i % CH) * 8, C::HALF));
            if (key0 + row >= most) {
              *y = make_uint4(0, 0, 0, 0);
            } else {
              constexpr uint32_t EL = Bits16<T>::kInf, EH = EL << 16;
              const uint32_t u[4] = {y->x, y->y, y->z, y->w};
#pragma unroll
              for (int k = 0; k < 4; ++k) bad |= (u[k] & EL) == EL || (u[k] & EH) == EH;
            }
          }
          fence_async_smem();                                // the next copy into this place comes after these writes
          bad = __any_sync(0xffffffffu, bad);
        }
        bool raise = false;
        float alpha[MT][2];
#pragma unroll
        for (int t = 0; t < MT; ++t)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = fmaxf(fmaxf(x[t][0][2 * e], x[t][0][2 * e + 1]), fmaxf(x[t][1][2 * e], x[t][1][2 * e + 1]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)) * c;
            // the maximum only moves when it grows by more than 2^8
            const bool need = mx > m[t][e] + 8.f;
            const float mn = need ? mx : m[t][e];
            alpha[t][e] = ex2(m[t][e] - mn);
            raise |= need;
            m[t][e] = mn;
            float sum = 0.f;
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int i = 2 * e; i < 2 * e + 2; ++i) {
                x[t][n][i] = ex2(fmaf(x[t][n][i], c, -mn));
                sum += x[t][n][i];
              }
            l[t][e] = fmaf(l[t][e], alpha[t][e], sum);
          }
        if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i) o[t][n][i] *= alpha[t][i >> 1];
        }
        if (!bad) {
          // the weights are rounded to the tensors' type for the product with V;
          // their sum is of the unrounded ones
          uint32_t a[MT][4];
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            a[t][0] = pack2<T>(x[t][0][0], x[t][0][1]);
            a[t][1] = pack2<T>(x[t][0][2], x[t][0][3]);
            a[t][2] = pack2<T>(x[t][1][0], x[t][1][1]);
            a[t][3] = pack2<T>(x[t][1][2], x[t][1][3]);
          }
#pragma unroll
          for (int n = 0; n < D / 16; ++n) {
            uint32_t b[4];
            ldsm4_t(vs + (n >> 2) * C::HALF + vrow * 128 + ((((n & 3) * 2 + vcol) ^ (vrow & 7)) << 4), b);
#pragma unroll
            for (int t = 0; t < MT; ++t) {
              mma16816<T>(o[t][2 * n], a[t], b[0], b[1]);
              mma16816<T>(o[t][2 * n + 1], a[t], b[2], b[3]);
            }
          }
        } else {
          // a NaN or infinity that only some rows may see: row by row on the CUDA cores
          float* w = reinterpret_cast<float*>(smem + C::MERGE + C::WEIGHTS) + warp * R * 16;
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int i = 0; i < 4; ++i) w[(t * 16 + (i >> 1) * 8 + qr) * 16 + n * 8 + qc + (i & 1)] = x[t][n][i];
          __syncwarp();
          const unsigned char* v = smem + st * 2 * C::TILE + C::TILE;
#pragma unroll 1
          for (int k = 0; k < 16; ++k) {
#pragma unroll
            for (int n = 0; n < D / 8; ++n) {
              const float2 f =
                  unpack2<T>(*reinterpret_cast<const uint32_t*>(v + swizzled(warp * 16 + k, n * 8 + qc, C::HALF)));
#pragma unroll
              for (int t = 0; t < MT; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                  if (key0 + k < limit[t][e]) {
                    const float pw = w[(t * 16 + e * 8 + qr) * 16 + k];
                    o[t][n][2 * e] = fmaf(pw, f.x, o[t][n][2 * e]);
                    o[t][n][2 * e + 1] = fmaf(pw, f.y, o[t][n][2 * e + 1]);
                  }
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(EMPTY(st));
      }
      // ---- the four warps' results together, in their order ----
      team_sync();                                           // the space has been read as Q
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 1);
          l[t][e] += __shfl_xor_sync(0xffffffffu, l[t][e], 2);
          if ((lane & 3) == 0) reinterpret_cast<float2*>(merge)[warp * R + t * 16 + e * 8 + qr] = make_float2(m[t][e], l[t][e]);
        }
      team_sync();
      const bool whole = s.whole();
      Slot<D, 32>& slot = static_cast<Slot<D, 32>*>(maps.partial)[2 * blockIdx.x + (s.a == 0 ? 1 : 0)];
      float f[MT][2];                                        // this warp's factor of each row
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = t * 16 + e * 8 + qr;
          float top = kNoMax, sum = 0.f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) top = fmaxf(top, reinterpret_cast<float2*>(merge)[w * R + r].x);
#pragma unroll
          for (int w = 0; w < kWarps; ++w) {
            const float2 ml = reinterpret_cast<float2*>(merge)[w * R + r];
            sum = fmaf(ml.y, ex2(ml.x - top), sum);
          }
          f[t][e] = ex2(m[t][e] - top);
          if (whole) f[t][e] *= sum == 0.f ? 0.f : 1.f / sum;
          else if (warp == 0 && (lane & 3) == 0) slot.ml[r] = make_float2(top, sum);
        }
      team_sync();
      // R x D, the 8-column blocks of row r turned by r so that a fragment's rows meet different banks
#pragma unroll 1
      for (int w = 0; w < kWarps; ++w) {
        if (warp == w) {
#pragma unroll
          for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int r = t * 16 + e * 8 + qr;
#pragma unroll
              for (int n = 0; n < D / 8; ++n) {
                float2* at = reinterpret_cast<float2*>(merge + r * D + ((n + r) % (D / 8)) * 8 + qc);
                const float2 was = w ? *at : make_float2(0.f, 0.f);
                *at = make_float2(fmaf(o[t][n][2 * e], f[t][e], was.x), fmaf(o[t][n][2 * e + 1], f[t][e], was.y));
              }
            }
        }
        team_sync();
      }
      for (int i = threadIdx.x; i < R * (D / 8); i += 32 * kWarps) {
        const int r = whole ? i / (D / 8) : i % R, n = whole ? i % (D / 8) : i / R;
        const int tok = r / p.group, g = r - tok * p.group;
        if (tok >= ntok) continue;
        const float4* at = reinterpret_cast<const float4*>(merge + r * D + ((n + r) % (D / 8)) * 8);
        const float4 a = at[0], b = at[1];
        if (whole) {
          *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (int64_t)(s.r.first + tok0 + tok) * p.o_ts +
                                    (int64_t)(s.h * p.group + g) * p.o_hs + n * 8) =
              make_uint4(pack2<T>(a.x, a.y), pack2<T>(a.z, a.w), pack2<T>(b.x, b.y), pack2<T>(b.z, b.w));
        } else {
          *reinterpret_cast<float4*>(slot.o[2 * n][r]) = a;
          *reinterpret_cast<float4*>(slot.o[2 * n + 1][r]) = b;
        }
      }
      team_sync();
    }
  }
#undef FULL
#undef EMPTY
}

static int64_t begun_bytes(int blocks) { return ((int64_t)blocks * (int64_t)sizeof(Begun) + 15) / 16 * 16; }

template <typename T, int D, int MT>
static int launch(const char* what, const Params& p, void* workspace, cudaStream_t stream) {
  using C = Cfg<D, MT>;
  Maps maps;
  if (!kv_maps(p, IsBf16<T>::v, kKeys, &maps.k, &maps.v, &maps.box)) {
    set_error("%s: cuTensorMapEncodeTiled failed", what);
    return JO_ERR_CUDA;
  }
  const int blocks = kBlocksPerSm * sm_count();
  maps.tpi = C::R / p.group;
  // no item has a cut inside when none is long enough to have one away from its edges
  const bool split = (int64_t)p.width * p.page > (2 * kMin - 1) * kKeys;
  maps.begun = split ? static_cast<Begun*>(workspace) : nullptr;
  maps.partial = static_cast<char*>(workspace) + begun_bytes(blocks);
  static bool attr[kMaxDevices] = {};
  const int dev = device_slot();
  if (!attr[dev]) {
    if (cudaFuncSetAttribute(few_kernel<T, D, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::BYTES) != cudaSuccess)
      return check_launch(what);
    attr[dev] = true;
  }
  few_kernel<T, D, MT><<<blocks, kThreads, C::BYTES, stream>>>(maps, p);
  if (split) launch_join<T, D, 32, C::R, 8>(p, maps.partial, maps.begun, maps.tpi, blocks, stream);
  return check_launch(what);
}

template <typename T, int D>
static int launch_rows(const char* what, const Params& p, int64_t rows, void* workspace, cudaStream_t stream) {
  return rows <= 16 ? launch<T, D, 1>(what, p, workspace, stream) : launch<T, D, 2>(what, p, workspace, stream);
}

}  // namespace few

int64_t few_workspace(int head_dim) {
  const int n = few::kBlocksPerSm * sm_count();
  return few::begun_bytes(n) + 2 * (int64_t)n * (int64_t)(head_dim == 64 ? sizeof(Slot<64, 32>) : sizeof(Slot<128, 32>));
}

int launch_few(const char* what, const Params& p, int64_t rows, int dtype, void* workspace, cudaStream_t s) {
  if (dtype == JO_DTYPE_BF16)
    return p.head_dim == 64 ? few::launch_rows<__nv_bfloat16, 64>(what, p, rows, workspace, s)
                            : few::launch_rows<__nv_bfloat16, 128>(what, p, rows, workspace, s);
  return p.head_dim == 64 ? few::launch_rows<__half, 64>(what, p, rows, workspace, s)
                          : few::launch_rows<__half, 128>(what, p, rows, workspace, s);
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
