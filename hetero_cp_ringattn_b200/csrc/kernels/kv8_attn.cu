// Attention over the paged 8-bit KV cache for a few query tokens per request (decode, drafts).
//
//   o = softmax(scale q K^T) V over the request's cached rows, K = ks[page] Kc, V = vs[page] Vc
//
// Query token i of a request with n cached rows and m query tokens sees rows 0 .. n - m + i; a row
// that sees nothing gives o = 0, lse = -inf.
//
// Bound: the cache bytes (2 Hkv D a cached token, read once); a GQA group has at most a few query
// rows, far below tcgen05's tile, so the products run on warp-level m16n8k16 f16 MMAs with the
// roles swapped: S^T = K Q^T and O^T = V^T P^T, the cached tokens (or head dims) on the 16-row side
// and up to 8 query rows a column tile, half the MMAs and accumulators that 16 padded query rows
// would take. 8-bit codes convert to f16 exactly, so K and V enter the products unrounded:
//   K   scales multiply the 32-bit scores; q is brought to f16 range by a power of two per row.
//   V   the scale moves into the exponent: p = 2^(s + log2 vs - m + 15) with m the running maximum
//       of s + log2 vs, O += p Vc, l += p / vs. So one page's scale costs one addition a score, and
//       no accumulator is rescaled for it. The 2^15 puts p's f16 rounding (2^-11 relative) down to
//       2^-29 of the maximum and its last nonzero at 2^-39: long tails of small weights count.
// Softmax statistics and accumulators are float32.
//
// Work: tiles of 32 cached tokens. The tiles of all (request, KV head, query row tile) items form
// one list, cut into equal ranges, one per warp (8 warps a CTA, one CTA per SM): a ragged batch and
// one long request load every SM alike, and no warp waits for another. A warp streams its tiles
// through its own ring of TMA boxes (128- or 64-byte swizzle, conflict-free ldmatrix), page ids and
// scales looked up one tile ahead of the copies. An item inside one range is finished in registers;
// the pieces of the others are (m, l, O) partials that a second small launch combines in list order.
#include <cuda.h>
#include <cudaTypedefs.h>

#include "kv8_common.cuh"
#include "launch.h"

namespace hcp {
namespace kv8 {

using namespace hcp::dev;

namespace {

constexpr int kWarps = 8;
constexpr int kTile = 32;     // cached tokens a tile
constexpr float kShift = 15.f;
constexpr float kLn2 = 0.6931471805599453f;

template <int D>
struct Ring {
  static constexpr int kBytes = 2 * kTile * D;            // K and V of a tile
  static constexpr int kStages = D == 128 ? 3 : 6;        // 192 KB for the 8 warps
};

struct Layout {  // workspace
  long long* prefix;   // [B + 1] tiles before each request
  float* ml;           // [workers][2][rows][2]
  float* o;            // [workers][2][rows][D]
};

__host__ __device__ inline size_t align256(size_t n) { return (n + 255) & ~size_t(255); }

__host__ __device__ inline Layout layout_of(void* ws, int B, int workers, int rows) {
  char* p = reinterpret_cast<char*>(ws);
  Layout l;
  l.prefix = reinterpret_cast<long long*>(p);
  p += align256(size_t(B + 1) * sizeof(long long));
  l.ml = reinterpret_cast<float*>(p);
  p += align256(size_t(workers) * 2 * rows * 2 * sizeof(float));
  l.o = reinterpret_cast<float*>(p);
  return l;
}

__device__ __forceinline__ void tma_load_4d(void* dst, const void* map, uint64_t* bar, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(smem_u32(bar)), "r"(0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// 16-byte piece `chunk` of token row `tok` in a TMA box with the swizzle of its row length.
template <int D>
__device__ __forceinline__ uint32_t piece(int tok, int chunk) {
  return D == 128 ? uint32_t(tok * 128 + ((chunk ^ (tok & 7)) << 4))
                  : uint32_t(tok * 64 + ((chunk ^ ((tok >> 1) & 3)) << 4));
}

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ int q_tokens(const AttnArgs& a, int b, int& first) {
  if (a.cu == nullptr) {
    first = b;
    return 1;
  }
  first = max(a.cu[b], 0);
  return max(0, min(min(a.cu[b + 1], a.T) - first, a.max_q));
}

// Cached rows of request b, no more than its table row can hold.
__device__ __forceinline__ int rows_of(const AttnArgs& a, int b) {
  return int(min((long long)max(a.kv_len[b], 0), (long long)a.width * a.c.P));
}

// One warp's place in the tile list.
struct Place {
  int b, h, rt, tile, tiles;  // request, KV head, query row tile, tile and tiles of the item
};

// First worker whose range [w W / NW, (w + 1) W / NW) reaches past x.
__device__ __forceinline__ int worker_of(long long x, long long W, int NW) { return int(((x + 1) * NW - 1) / W); }

template <int D, int NT, bool INT8>
__global__ void __launch_bounds__(kWarps * 32, 1)
attn_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, AttnArgs a) {
  constexpr int kStages = Ring<D>::kStages, kBytes = Ring<D>::kBytes, kChunks = D / 16, kRows = 8 * NT;
  extern __shared__ unsigned char raw[];
  unsigned char* ring_base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  long long* prefix = reinterpret_cast<long long*>(ring_base + kWarps * kStages * kBytes);
  __shared__ uint64_t bars[kWarps][kStages];
  __shared__ float meta[kWarps][kStages][4];   // k scale and v scale of the tile's two halves
  __shared__ long long warp_tot[kWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = a.H / a.c.Hkv, P = a.c.P, Hkv = a.c.Hkv;
  if (tid == 0) {
    for (int w = 0; w < kWarps; ++w)
      for (int i = 0; i < kStages; ++i) mbar_init(&bars[w][i], 1);
    fence_barrier_init();
    tma_prefetch_desc(&kmap);
    tma_prefetch_desc(&vmap);
  }
  pdl_trigger();
  pdl_wait();

  // ---------------------------------------------------------------- the tile list
  {
    const int per = (a.B + kWarps * 32 - 1) / (kWarps * 32);
    const int r0 = min(a.B, tid * per), r1 = min(a.B, r0 + per);
    auto tiles_of = [&](int b) {
      int first;
      const int qn = q_tokens(a, b, first);
      return (long long)Hkv * ((qn * G + kRows - 1) / kRows) * ((rows_of(a, b) + kTile - 1) / kTile);
    };
    long long own = 0;
    for (int b = r0; b < r1; ++b) own += tiles_of(b);
    long long inc = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long up = __shfl_up_sync(0xffffffffu, inc, d);
      if (lane >= d) inc += up;
    }
    if (lane == 31) warp_tot[warp] = inc;
    __syncthreads();
    long long ex = inc - own;
    for (int w = 0; w < warp; ++w) ex += warp_tot[w];
    for (int b = r0; b < r1; ++b) {
      prefix[b] = ex;
      ex += tiles_of(b);
      if (b + 1 == a.B) prefix[a.B] = ex;
    }
    __syncthreads();
  }
  const int NW = gridDim.x * kWarps, worker = warp * gridDim.x + blockIdx.x;
  const Layout L = layout_of(a.workspace, a.B, NW, kRows);
  if (blockIdx.x == 0)
    for (int b = tid; b <= a.B; b += kWarps * 32) L.prefix[b] = prefix[b];
  const long long W = prefix[a.B];
  const long long x0 = W * worker / NW, x1 = W * (worker + 1) / NW;
  if (x0 >= x1) return;

  auto place_of = [&](long long x) {
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] <= x) lo = mid;
      else hi = mid;
    }
    Place p;
    p.b = lo;
    int first;
    const int rts = (q_tokens(a, lo, first) * G + kRows - 1) / kRows;
    p.tiles = (rows_of(a, lo) + kTile - 1) / kTile;
    const long long rem = x - prefix[lo];
    const int item = int(rem / p.tiles);
    p.tile = int(rem - (long long)item * p.tiles);
    p.h = item / rts;
    p.rt = item - p.h * rts;
    return p;
  };

  // ---------------------------------------------------------------- the copies' side
  unsigned char* ring = ring_base + warp * kStages * kBytes;
  // a tile lies in one page of 32 tokens or more, or in two of 16 (lane 1 brings the second half)
  const int halves = P == 16 ? 2 : 1;
  const int box = min(P, kTile);
  long long px = x0;          // next tile whose page is looked up
  Place pp = place_of(px);
  int next_page = -1, next_row = 0, next_h = 0;   // looked up, not yet copied
  bool next_valid = false;
  auto look_up = [&] {
    next_valid = false;
    if (px < x1) {
      const int block = pp.tile * kTile / P + lane;
      if (lane < halves && block * P < rows_of(a, pp.b)) {
        next_page = a.table[(long)pp.b * a.width + block];
        next_valid = true;
      }
      next_row = pp.tile * kTile % P;
      next_h = pp.h;
      ++px;
      if (++pp.tile == pp.tiles && px < x1) pp = place_of(px);
    }
  };
  float load_ks = 1.f, load_vs = 1.f;             // scales of the tile copied last
  int load_stage = -1;
  auto put_scales = [&] {
    if (load_stage >= 0 && lane < halves) {
      meta[warp][load_stage][2 * lane] = load_ks;
      meta[warp][load_stage][2 * lane + 1] = load_vs;
      if (halves == 1) {
        meta[warp][load_stage][2] = load_ks;
        meta[warp][load_stage][3] = load_vs;
      }
    }
    load_stage = -1;
  };
  auto copy = [&](int stage) {
    const uint32_t valid = __ballot_sync(0xffffffffu, next_valid);
    if (valid == 0) return;
    uint64_t* bar = &bars[warp][stage];
    if (lane == 0) mbar_arrive_expect_tx(bar, uint32_t(__popc(valid)) * 2u * uint32_t(box) * D);
    __syncwarp();
    load_ks = load_vs = 1.f;
    if (next_valid) {
      unsigned char* dst = ring + stage * kBytes + lane * 16 * D;
      // a page id outside the pool reads as zeros (the tensor map's bounds)
      tma_load_4d(dst, &kmap, bar, next_row, next_h, next_page);
      tma_load_4d(dst + kTile * D, &vmap, bar, next_row, next_h, next_page);
      if (next_page >= 0 && next_page < a.c.pages) {
        const long at = (long)next_page * a.c.scale_page_stride + (long)next_h * a.c.scale_head_stride;
        load_ks = a.c.k_scale[at];
        load_vs = a.c.v_scale[at];
      } else {
        report_error(a.status, int(StatusCode::kOutOfBounds), 411, next_page, next_h);
      }
    }
    load_stage = stage;
  };
  look_up();
#pragma unroll 1
  for (int i = 0; i < kStages; ++i) {
    put_scales();
    copy(i);
    look_up();
  }
  put_scales();
  __syncwarp();

  // ---------------------------------------------------------------- the products' side
  const int j = lane >> 2, c = lane & 3;   // fragment row and column group of the lane
  int stage = 0;
  uint32_t phase = 0;
  long long x = x0;
  bool alive = true;
  while (x < x1 && alive) {
    const Place p = place_of(x);
    const int n = rows_of(a, p.b);
    int first;
    const int qn = q_tokens(a, p.b, first);
    const int end = int(min((long long)p.tiles, p.tile + (x1 - x)));
    const int r0 = p.rt * kRows, rows = min(qn * G - r0, kRows);   // the item's query rows

    // q as the f16 B operand: lane (j, c) holds row j of each column tile, dims 16 s + 4 c .. + 3 of
    // k step s (the same order in which a lane's K bytes come out of ldmatrix)
    uint32_t qf[NT][kChunks][2];
    float f[NT][2];          // score factor of the lane's two columns
    int lim[NT][2];          // rows seen by them
    float m[NT][2], l[NT][2];
    float acc[kChunks][NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int r = t * 8 + j;
      float v[kChunks][4];
      float top = 0.f;
      const bool have = r < rows;
      const int qi = (r0 + r) / G, g = (r0 + r) % G;
      const uint16_t* src = reinterpret_cast<const uint16_t*>(a.q) + (long)(first + qi) * a.q_stride +
                            (long)(p.h * G + g) * a.q_head_stride + 4 * c;
#pragma unroll
      for (int s = 0; s < kChunks; ++s) {
        const uint2 w = have ? *reinterpret_cast<const uint2*>(src + 16 * s) : make_uint2(0, 0);
        if (a.q_dtype == kBF16) {
          v[s][0] = bf16_lo(w.x); v[s][1] = bf16_hi(w.x); v[s][2] = bf16_lo(w.y); v[s][3] = bf16_hi(w.y);
        } else {
          const float2 lo = half2_floats(w.x), hi = half2_floats(w.y);
          v[s][0] = lo.x; v[s][1] = lo.y; v[s][2] = hi.x; v[s][3] = hi.y;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, fabsf(v[s][i]));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // |q| 2^k in [2^14, 2^15) for the row's largest element
      const int e = top > 0.f ? max(-113, min(100, 14 - (((__float_as_int(top) >> 23) & 0xff) - 127))) : 0;
      const float up = pow2(e);
#pragma unroll
      for (int s = 0; s < kChunks; ++s) {
        qf[t][s][0] = pack_half(v[s][0] * up, v[s][1] * up);
        qf[t][s][1] = pack_half(v[s][2] * up, v[s][3] * up);
      }
      const float back = a.scale * 1.4426950408889634f * pow2(-e);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        f[t][i] = __shfl_sync(0xffffffffu, back, (2 * c + i) * 4);
        const int col = t * 8 + 2 * c + i;
        lim[t][i] = col < rows ? n - qn + (r0 + col) / G + 1 : n;
        m[t][i] = -INFINITY;
        l[t][i] = 0.f;
      }
#pragma unroll
      for (int s = 0; s < kChunks; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[s][t][i] = 0.f;
    }
    const int qi0 = r0 / G, qi1 = (r0 + rows - 1) / G;    // the item's query tokens
    const int least = n - qn + qi0 + 1;                   // rows that all of them see

    for (int tile = p.tile; tile < end; ++tile, ++x) {
      if (!mbar_wait(&bars[warp][stage], phase, a.status, 412)) {
        alive = false;
        break;
      }
      const int base = tile * kTile;
      const uint32_t kbase = smem_u32(ring + stage * kBytes), vbase = kbase + kTile * D;
      // ---- S^T = K Q^T
      float s[2][NT][4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[mt][t][i] = 0.f;
#pragma unroll
        for (int k = 0; k < kChunks; k += 2) {
          uint32_t r[4];
          ldmatrix4(kbase + piece<D>(mt * 16 + (lane & 15), k + (lane >> 4)), r);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t af[4];
            decode4<INT8>(r[2 * h], af[0], af[2]);
            decode4<INT8>(r[2 * h + 1], af[1], af[3]);
#pragma unroll
            for (int t = 0; t < NT; ++t) mma_f16(s[mt][t], af, qf[t][k + h][0], qf[t][k + h][1]);
          }
        }
      }
      // ---- scores in the log2 domain, masked, and the running maximum
      const bool edge = base + kTile > least;
      float lv[2], iv[2];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const float ks = meta[warp][stage][2 * mt], vs = meta[warp][stage][2 * mt + 1];
        // a block scaled by 0 holds zeros: its weight counts in l and its p V is 0 whatever p is
        lv[mt] = vs > 0.f ? __log2f(vs) : 0.f;
        iv[mt] = vs > 0.f ? __fdividef(1.f, vs) : 1.f;
        if (!(vs == vs)) lv[mt] = vs;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float v = fmaf(s[mt][t][i], f[t][i & 1] * ks, lv[mt]);
            if (edge && base + mt * 16 + j + (i >> 1) * 8 >= lim[t][i & 1]) v = -INFINITY;
            s[mt][t][i] = v;
          }
      }
      float up[NT][2], mu[NT][2];
      bool changed = false;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float v = fmaxf(fmaxf(s[0][t][i], s[0][t][i + 2]), fmaxf(s[1][t][i], s[1][t][i + 2]));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
          const float now = fmaxf(m[t][i], v);
          mu[t][i] = (now == -INFINITY ? 0.f : now) - kShift;
          up[t][i] = fast_exp2(m[t][i] - kShift - mu[t][i]);
          changed |= now > m[t][i];
          m[t][i] = now;
        }
      if (__any_sync(0xffffffffu, changed)) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
          for (int k = 0; k < kChunks; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[k][t][i] *= up[t][i & 1];
          l[t][0] *= up[t][0];
          l[t][1] *= up[t][1];
        }
      }
      // ---- p, its sum, and P^T as the B operand
      uint32_t pf[2][NT][2];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const float vs = meta[warp][stage][2 * mt + 1];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float e[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            e[i] = fast_exp2(s[mt][t][i] - mu[t][i & 1]);
            l[t][i & 1] = fmaf(e[i], iv[mt], l[t][i & 1]);
          }
          if (vs == 0.f) e[0] = e[1] = e[2] = e[3] = 0.f;
          pf[mt][t][0] = transpose8x8(pack_half(e[0], e[1]));
          pf[mt][t][1] = transpose8x8(pack_half(e[2], e[3]));
        }
      }
      // ---- O^T += V^T P^T. In a tile that ends inside the rows some query token sees, every query
      // token gets a pass of its own with the codes it must not see taken as 0: whatever a masked
      // place holds (stale bytes behind the end, NaN in a later draft's row), p = 0 cannot cancel it.
      auto values = [&](int seen, bool all) {
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          uint32_t b0[NT], b1[NT];
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            // column j of the operand is query row t * 8 + j: only this pass's rows
            const bool mine = all || (n - qn + (r0 + t * 8 + j) / G + 1) == seen;
            b0[t] = mine ? pf[mt][t][0] : 0u;
            b1[t] = mine ? pf[mt][t][1] : 0u;
          }
          const int tok = base + mt * 16 + 2 * c;
#pragma unroll
          for (int k = 0; k < kChunks; k += 2) {
            uint32_t r[4];
            ldmatrix4_trans(vbase + piece<D>(mt * 16 + (lane & 15), k + (lane >> 4)), r);
            if (!all) {
              // a register holds two codes of token 2 c (low half) and two of token 2 c + 1
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int at = tok + (i & 1) * 8;
                r[i] &= (at < seen ? 0xffffu : 0u) | (at + 1 < seen ? 0xffff0000u : 0u);
              }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t af[4];
              decode4<INT8>(__byte_perm(r[2 * h], 0, 0x3120), af[0], af[1]);
              decode4<INT8>(__byte_perm(r[2 * h + 1], 0, 0x3120), af[2], af[3]);
#pragma unroll
              for (int t = 0; t < NT; ++t) mma_f16(acc[k + h][t], af, b0[t], b1[t]);
            }
          }
        }
      };
      if (!edge) {
        values(0, true);
      } else {
#pragma unroll 1
        for (int qi = qi0; qi <= qi1; ++qi) {
          const int seen = n - qn + qi + 1;
          if (seen > base) values(seen, false);
        }
      }
      // ---- the stage is free: scales and copy of the tile kStages ahead, look-up of the one after
      __syncwarp();
      put_scales();
      copy(stage);
      look_up();
      if (++stage == kStages) {
        stage = 0;
        phase ^= 1;
      }
    }
    // copies look up and write one tile late: the last scales of a finished range are never read
    // ---------------------------------------------------------------- the item's result
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float v = l[t][i];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        v += __shfl_xor_sync(0xffffffffu, v, 16);
        l[t][i] = v;
      }
    const bool complete = p.tile == 0 && end == p.tiles;
    if (complete) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = t * 8 + 2 * c + i;
          if (r < rows) {
            const int qi = (r0 + r) / G, head = p.h * G + (r0 + r) % G;
            const float inv = l[t][i] == 0.f ? 0.f : __frcp_rn(l[t][i]);
            uint32_t* o = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.o) + ((long)(first + qi) * a.H + head) * D);
#pragma unroll
            for (int k = 0; k < kChunks; ++k) o[k * 8 + j] = pack16(a.q_dtype, acc[k][t][i] * inv, acc[k][t][i + 2] * inv);
            if (j == 0 && a.lse != nullptr)
              a.lse[(long)head * a.T + first + qi] = l[t][i] == 0.f ? -INFINITY : (m[t][i] - kShift + log2f(l[t][i])) * kLn2;
          }
        }
    } else {
      // slot 0: the piece starts the worker's range; slot 1: it starts the item
      const int slot = (x - (end - p.tile) == x0) ? 0 : 1;
      float* po = L.o + ((size_t)worker * 2 + slot) * kRows * D;
      float* pm = L.ml + ((size_t)worker * 2 + slot) * kRows * 2;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = t * 8 + 2 * c + i;
          if (r < rows) {
            float2* o = reinterpret_cast<float2*>(po + (size_t)r * D);
#pragma unroll
            for (int k = 0; k < kChunks; ++k) o[k * 8 + j] = make_float2(acc[k][t][i], acc[k][t][i + 2]);
            if (j == 0) *reinterpret_cast<float2*>(pm + 2 * r) = make_float2(m[t][i], l[t][i]);
          }
        }
    }
  }
}

// One CTA per (query token, head): the pieces of its item in list order, (m, l, O) each.
constexpr int kCombineWarps = 4;

template <int D, int NT>
__global__ void __launch_bounds__(kCombineWarps * 32) combine_kernel(AttnArgs a, int NW) {
  constexpr int kRows = 8 * NT, kPer = D / 32;
  __shared__ float part[kCombineWarps][D];
  __shared__ float part_l[kCombineWarps];
  pdl_trigger();
  pdl_wait();
  const int t = blockIdx.x / a.H, head = blockIdx.x % a.H;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int G = a.H / a.c.Hkv;
  // the token's request
  int b = t;
  if (a.cu != nullptr) {
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (a.cu[mid] <= t) lo = mid;
      else hi = mid;
    }
    b = lo;
  }
  int first;
  const int qn = q_tokens(a, b, first);
  const int qi = t - first;
  const Layout L = layout_of(a.workspace, a.B, NW, kRows);
  const int n = rows_of(a, b);
  const int tiles = (n + kTile - 1) / kTile;
  uint16_t* out = reinterpret_cast<uint16_t*>(a.o) + ((long)t * a.H + head) * D;
  if (qi < 0 || qi >= qn || tiles == 0) {   // no cached rows (or a token outside every request)
    if (threadIdx.x < D / 2) reinterpret_cast<uint32_t*>(out)[threadIdx.x] = 0u;
    if (threadIdx.x == 0 && a.lse != nullptr) a.lse[(long)head * a.T + t] = -INFINITY;
    return;
  }
  const int rts = (qn * G + kRows - 1) / kRows;
  const int r = qi * G + head % G, rt = r / kRows;
  const long long W = L.prefix[a.B];
  const long long start = L.prefix[b] + ((long long)(head / G) * rts + rt) * tiles, stop = start + tiles;
  const int w0 = worker_of(start, W, NW), w1 = worker_of(stop - 1, W, NW);
  if (w0 == w1) return;                     // finished by its only worker
  const int row = r - rt * kRows;
  // with fewer tiles than workers some ranges in between are empty
  auto empty = [&](int w) { return W * w / NW == W * (w + 1) / NW; };
  auto slot_of = [&](int w) { return (size_t)w * 2 + ((w == w0 && start > W * w / NW) ? 1 : 0); };
  float top = -INFINITY;
  for (int w = w0 + lane; w <= w1; w += 32)
    if (!empty(w)) top = fmaxf(top, L.ml[(slot_of(w) * kRows + row) * 2]);
  top = warp_max(top);
  const float base = top == -INFINITY ? 0.f : top;
  float acc[kPer], l = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) acc[i] = 0.f;
#pragma unroll 4
  for (int w = w0 + warp; w <= w1; w += kCombineWarps) {
    if (empty(w)) continue;
    const size_t at = slot_of(w) * kRows + row;
    const float2 ml = *reinterpret_cast<const float2*>(L.ml + at * 2);
    const float e = fast_exp2(ml.x - base);
    l = fmaf(e, ml.y, l);
    const float* o = L.o + at * D + lane * kPer;
#pragma unroll
    for (int i = 0; i < kPer; i += 2) {
      const float2 v = *reinterpret_cast<const float2*>(o + i);
      acc[i] = fmaf(e, v.x, acc[i]);
      acc[i + 1] = fmaf(e, v.y, acc[i + 1]);
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) part[warp][lane * kPer + i] = acc[i];
  if (lane == 0) part_l[warp] = l;
  __syncthreads();
  l = 0.f;
  for (int w = 0; w < kCombineWarps; ++w) l += part_l[w];
  if (threadIdx.x < D / 2) {
    float v0 = 0.f, v1 = 0.f;
#pragma unroll
    for (int w = 0; w < kCombineWarps; ++w) {
      v0 += part[w][2 * threadIdx.x];
      v1 += part[w][2 * threadIdx.x + 1];
    }
    const float inv = l == 0.f ? 0.f : __frcp_rn(l);
    reinterpret_cast<uint32_t*>(out)[threadIdx.x] = pack16(a.q_dtype, v0 * inv, v1 * inv);
  }
  if (threadIdx.x == 0 && a.lse != nullptr)
    a.lse[(long)head * a.T + t] = l == 0.f ? -INFINITY : (top - kShift + log2f(l)) * kLn2;
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  return fn;
}

// [pages][Hkv][P][D] bytes; a box is up to 32 tokens of one (page, head).
bool make_map(CUtensorMap* map, const uint8_t* base, const Cache& c) {
  const cuuint64_t dims[4] = {cuuint64_t(c.D), cuuint64_t(c.P), cuuint64_t(c.Hkv), cuuint64_t(c.pages)};
  const cuuint64_t strides[3] = {cuuint64_t(c.token_stride), cuuint64_t(c.head_stride), cuuint64_t(c.page_stride)};
  const cuuint32_t box[4] = {cuuint32_t(c.D), cuuint32_t(c.P < kTile ? c.P : kTile), 1, 1};
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  return encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, const_cast<uint8_t*>(base), dims, strides, box, ones,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, c.D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Query rows of an item: 8 where a request's rows fit, else 16 (each tile's codes are converted
// once for both column tiles).
int column_tiles(const AttnArgs& a) { return a.max_q * (a.H / a.c.Hkv) <= 8 ? 1 : 2; }

template <int D, int NT, bool INT8>
cudaError_t launch_attn(const AttnArgs& a, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t s) {
  const int grid = a.num_sms;
  const size_t smem = 1024 + size_t(kWarps) * Ring<D>::kStages * Ring<D>::kBytes + size_t(a.B + 1) * sizeof(long long);
  auto kernel = attn_kernel<D, NT, INT8>;
  cudaError_t e = once_per_device_kernel(reinterpret_cast<const void*>(kernel), [&] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                int(1024 + size_t(kWarps) * Ring<D>::kStages * Ring<D>::kBytes + (kAttnMaxRows + 1) * sizeof(long long)));
  });
  if (e != cudaSuccess) return e;
  e = launch_pdl(kernel, dim3(unsigned(grid)), dim3(kWarps * 32), smem, s, km, vm, a);
  if (e != cudaSuccess) return e;
  return launch_pdl(combine_kernel<D, NT>, dim3(unsigned(a.T) * unsigned(a.H)), dim3(kCombineWarps * 32), 0, s, a, grid * kWarps);
}

template <int D, int NT>
cudaError_t attn_code(const AttnArgs& a, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t s) {
  return a.c.code == kInt8 ? launch_attn<D, NT, true>(a, km, vm, s) : launch_attn<D, NT, false>(a, km, vm, s);
}

}  // namespace

size_t attention_workspace(const AttnArgs& a) {
  const size_t workers = size_t(a.num_sms) * kWarps, rows = 8 * size_t(column_tiles(a));
  return align256(size_t(a.B + 1) * sizeof(long long)) + align256(workers * 2 * rows * 2 * sizeof(float)) +
         workers * 2 * rows * a.c.D * sizeof(float);
}

const char* attention(const AttnArgs& a, cudaStream_t s) {
  const Cache& c = a.c;
  if (c.D != 64 && c.D != 128) return "attention_kv8: head_dim must be 64 or 128";
  if (c.P != 16 && c.P != 32 && c.P != 64 && c.P != 128) return "attention_kv8: page must be 16, 32, 64 or 128 tokens";
  if (a.H < 1 || c.Hkv < 1 || a.H % c.Hkv) return "attention_kv8: heads must be a multiple of the KV heads";
  if (a.B > kAttnMaxRows) return "attention_kv8: at most 2048 requests";
  if ((long)a.T * a.H > 0x7fffffffl || (long)a.max_q * a.H > 0x3fffffffl || (long)a.width * c.P > 0x7fffffc0l)
    return "attention_kv8: too many query rows or cached rows";
  if (c.page_stride % 16 || c.head_stride % 16 || c.token_stride % 16 || reinterpret_cast<uintptr_t>(c.k) % 16 ||
      reinterpret_cast<uintptr_t>(c.v) % 16)
    return "attention_kv8: cache rows must start on 16-byte boundaries";
  if (a.q_stride % 4 || a.q_head_stride % 4 || reinterpret_cast<uintptr_t>(a.q) % 8)
    return "attention_kv8: q rows must start on 8-byte boundaries";
  if (a.T < 1 || a.B < 1) return nullptr;
  if (encode_fn() == nullptr) return "attention_kv8: cuTensorMapEncodeTiled is not available";
  CUtensorMap km, vm;
  if (!make_map(&km, c.k, c) || !make_map(&vm, c.v, c)) return "attention_kv8: the cache's strides do not make a tensor map";
  const int nt = column_tiles(a);
  cudaError_t e;
  if (c.D == 64) e = nt == 1 ? attn_code<64, 1>(a, km, vm, s) : attn_code<64, 2>(a, km, vm, s);
  else e = nt == 1 ? attn_code<128, 1>(a, km, vm, s) : attn_code<128, 2>(a, km, vm, s);
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace kv8
}  // namespace hcp
