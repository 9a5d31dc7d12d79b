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
//   K   scales multiply the 32-bit scores; q is brought to f16 range by a power of two per item (the
//       query rows of one request that share a KV head): bf16's 8 bits stay exact down to 2^-31 of the
//       item's largest element, f16's 11 to 2^-28, and below the error is 2^-39 of it.
//   V   the scale moves into the exponent: p = 2^(s + log2 vs - m + 15) with m the running maximum
//       of s + log2 vs, O += p Vc, l += p / vs. So one page's scale costs one addition a score, and
//       no accumulator is rescaled for it. The 2^15 puts p's f16 rounding (2^-11 relative) down to
//       2^-29 of the maximum and its last nonzero at 2^-39: long tails of small weights count.
// Softmax statistics and accumulators are float32.
//
// Work: tiles of 32 cached tokens. The tiles of all (request, KV head, query row tile) items form
// one list, cut into equal ranges, one a CTA (one CTA per SM) and within it one a stream: a ragged
// batch and one long request load every SM alike. A stream, a warp or a team of two, runs its tiles
// through its own ring of TMA boxes (128- or 64-byte swizzle, conflict-free ldmatrix); page ids are
// looked up one turn ahead of the copies, scales come with them. An item inside one range is finished
// in registers; a CTA's pieces are merged in shared memory, and an item that goes on in the next CTA
// is left as (m, l, O) partials that a second small launch combines in list order.
//
// Measured on B200, caches cold, cache bytes a second (a plain copy: 6.55 TB/s): 64 requests of up to
// 32768 rows, 8 KV heads of 128 dims, 4 query rows each: 222 us, 5.8 TB/s e4m3, 6.1 int8; 64 dims: 140
// us, 4.7. Small work is latency: one request of 4097 rows 15 us, of 131071 rows 32 us, 33 requests of
// up to 8192 44 to 48 us (some SMs, those of the larger clusters of SMs, end up to 10% later than
// others). Five tokens of 7 heads (35 rows): 299 us, where 100 are the bytes: bound by the chain from
// scores to weights to the next products with 8 warps an SM, the tensor cores 38% busy.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "kv8_common.cuh"
#include "launch.h"

namespace hcp {
namespace kv8 {

using namespace hcp::dev;

namespace {

constexpr int kTile = 32;     // cached tokens a tile
constexpr float kShift = 15.f;
constexpr float kNone = -3e38f;   // the running maximum before any score (finite: differences stay numbers)
constexpr float kLn2 = 0.6931471805599453f;

// How the warps of a CTA share the tile streams. kTeam warps work on a stream, kStep tiles at a time:
// each computes the scores of kMt 16-token groups, they exchange the column maxima and P, and each
// accumulates kOut 16-dim pieces of O over all tokens of the step. So up to 40 query rows take one pass
// over the cache with their accumulators in registers, no code is converted twice, and registers
// allow the warps that hide each other's latencies (a warp alone issues about every fifth cycle).
// 12 warps where registers allow it. 35 rows of 128 dims: 299 us; in single warps of 16 rows, three
// passes over the cache, 302 (and 2 times the memory traffic); in teams of four, 16 warps, 404.
// Arithmetic on pairs of columns (f32x2): 21 rows 214 -> 206 us, 35 rows 302 -> 299.
template <int D, int NT>
struct Shape {
  static constexpr int kTeam = NT <= 2 ? 1 : 2;
  static constexpr int kStep = NT <= 2 ? 1 : 2;
  static constexpr int kWarps = NT == 1 || (NT == 2 && D == 64) ? 12 : 8;
  static constexpr int kThreads = kWarps * 32;
  static constexpr int kRows = 8 * NT;                      // query rows of an item
  static constexpr int kStreams = kWarps / kTeam;
  static constexpr int kMt = 2 * kStep / kTeam;
  static constexpr int kOut = D / 16 / kTeam;
  static constexpr int kBytes = 2 * kTile * D;              // K and V of a tile
  // a team reads q's fragments from shared memory (80 registers a lane for 40 rows of 128 dims)
  static constexpr int kQBytes = kTeam > 1 ? kStreams * kRows * D * 2 : 0;
  static constexpr int kStages = ((kTeam > 1 ? 176 : 192) * 1024 - kQBytes) / (kStreams * kBytes);
  static constexpr int kRing = kStages * kBytes;
  static_assert(kMt >= 1 && kOut >= 2 && kOut % 2 == 0 && kStages >= 2 * kStep, "shape");
  static_assert(kRing >= kRows * D * 4, "a stream's last piece is left in its ring");
};

// An item (request, KV head, query row tile) that goes on in the next CTA.
struct __align__(16) Straddle {
  int last;            // the last CTA that works on it; -1: none
  int row0, rows;      // its query rows (token * G + head of the group, within the request)
  int first;           // the request's first query token
  int head;            // first query head of the KV head
  int pad[3];
};

struct Workspace {
  Straddle* straddle;  // [CTAs]
  float* ml;           // [CTAs][2][rows][2]   piece 0: of the item at the range's start; 1: at its end
  float* o;            // [CTAs][2][rows][D]
  float* head;         // [CTAs][streams][rows][D]  first pieces of streams that go on with another item
  size_t bytes;
};

__host__ __device__ inline size_t align256(size_t n) { return (n + 255) & ~size_t(255); }

__host__ __device__ inline Workspace workspace_of(void* ws, int ctas, int streams, int rows, int D) {
  char* p = reinterpret_cast<char*>(ws);
  Workspace w;
  w.straddle = reinterpret_cast<Straddle*>(p);
  size_t at = align256(size_t(ctas) * sizeof(Straddle));
  w.ml = reinterpret_cast<float*>(p + at);
  at += align256(size_t(ctas) * 2 * rows * 2 * sizeof(float));
  w.o = reinterpret_cast<float*>(p + at);
  at += align256(size_t(ctas) * 2 * rows * D * sizeof(float));
  w.head = reinterpret_cast<float*>(p + at);
  at += align256(size_t(ctas) * streams * rows * D * sizeof(float));
  w.bytes = at;
  return w;
}

// 64-bit quotient, by 32-bit division where both fit.
__device__ __forceinline__ long long quotient(long long x, long long y) {
  return ((x | y) >> 32) == 0 ? (long long)(uint32_t(x) / uint32_t(y)) : x / y;
}

// The tile list in `n` equal ranges: part i starts at begin(i).
struct Split {
  long long q, r;
  __device__ __forceinline__ Split(long long total, int n) : q(quotient(total, n)), r(total - q * n) {}
  __device__ __forceinline__ long long begin(int i) const { return q * i + min((long long)i, r); }
  __device__ __forceinline__ int part_of(long long x) const {   // the part that holds x
    const long long big = r * (q + 1);
    return int(x < big ? quotient(x, q + 1) : r + quotient(x - big, q));
  }
};

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

// (a call: inlined, 8 requests of up to 4096 rows took 16.8 us instead of 16.6)
__device__ __noinline__ void offsets_out_of_range(int* status, int to, int b) {
  report_error(status, int(StatusCode::kOutOfBounds), 413, to, b);
}

__device__ __forceinline__ int q_tokens(const AttnArgs& a, int b, int& first) {
  if (a.cu == nullptr) {
    first = b;
    return 1;
  }
  const int from = a.cu[b], to = a.cu[b + 1];
  first = max(from, 0);
  const int n = max(0, min(to, a.T) - first);
  // tokens that q does not hold would move the causal limits of those it holds
  if (n != to - from) offsets_out_of_range(a.status, to, b);
  return n;
}

// Cached rows of request b, no more than its table row can hold.
__device__ __forceinline__ int rows_of(const AttnArgs& a, int b) {
  return int(min((long long)max(a.kv_len[b], 0), (long long)a.width * a.c.P));
}

// A place in the tile list.
struct Place {
  int b, h, rt, tile, tiles;  // request, KV head, query row tile, tile and tiles of the item
  int n, qn, first;           // the request's cached rows, query tokens and the first of them
};

// A copying lane's next page, and its place in the list.
struct CopyLane {
  long long px;
  Place pp;
  int page, row, h;     // looked up: page id, first row in the page, KV head
  int tile, valid;      // there is a tile; it reaches into this page
};

__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}

// A finished row: o = acc / l, lse = (m - 15 + log2 l) ln 2; l = 0: the row saw nothing.
__device__ __forceinline__ float row_lse(float m, float l) { return l == 0.f ? -INFINITY : (m - kShift + log2f(l)) * kLn2; }
__device__ __forceinline__ float row_inv(float l) { return l == 0.f ? 0.f : __frcp_rn(l); }

// The warps of a stream meet (named barrier 1 + stream).
template <int TEAM>
__device__ __forceinline__ void team_sync(int stream) {
  if (TEAM == 1) __syncwarp();
  else asm volatile("bar.sync %0, %1;" ::"r"(stream + 1), "n"(32 * TEAM) : "memory");
}

template <int D, int NT, bool INT8>
__global__ void __launch_bounds__(Shape<D, NT>::kThreads, 1)
attn_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, AttnArgs a) {
  using S = Shape<D, NT>;
  constexpr int kTeam = S::kTeam, kWarps = S::kWarps, kMt = S::kMt, kOut = S::kOut;
  constexpr bool kShared = kTeam > 1;                      // q, maxima and P pass through shared memory
  constexpr int kStages = S::kStages, kBytes = S::kBytes, kRows = S::kRows, kStreams = S::kStreams, kStep = S::kStep;
  constexpr int kChunks = D / 16;                          // 16-dim pieces of a row
  extern __shared__ unsigned char raw[];
  unsigned char* ring_base = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  uint2* q_frag = reinterpret_cast<uint2*>(ring_base + kStreams * S::kRing);   // team: [stream][piece][tile][lane]
  long long* prefix = reinterpret_cast<long long*>(ring_base + kStreams * S::kRing + S::kQBytes);
  int* s_rows = reinterpret_cast<int*>(prefix + a.B + 1);    // cached rows of each request
  int* s_first = s_rows + a.B;                               // its first query token, and (next B) their number
  __shared__ uint64_t bars[kStreams][kStages];
  __shared__ float meta[kStreams][kStages][2][2];          // k scale and v scale of the tile's (two) pages
  __shared__ CopyLane s_copy[kStreams][2 * kStep];
  __shared__ long long warp_tot[kWarps];
  __shared__ float s_ml[kStreams][2][kRows][2];            // (m, l) of the streams' pieces
  __shared__ long long s_start[kStreams][2];               // first tile of the piece's item; -1: no piece
  __shared__ Place s_place[kStreams][2];
  __shared__ float s_max[kShared ? kStreams : 1][kTeam][kRows];   // team: the warps' column maxima
  __shared__ uint2 s_p[kShared ? kStreams : 1][2 * kStep][kShared ? NT : 1][32];   // team: P^T of each 16 tokens
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int stream = warp / kTeam, sub = warp % kTeam;
  const int G = a.H / a.c.Hkv, P = a.c.P, Hkv = a.c.Hkv;
  // a tile lies in one page of 32 tokens or more, or in two of 16
  const int halves = P == 16 ? 2 : 1;
  if (tid == 0) {
    // a stage is full with its pages' bytes and scales (a page's lane announces the bytes before it
    // arrives with the scales, so the count cannot complete ahead of them)
    for (int w = 0; w < kStreams; ++w)
      for (int i = 0; i < kStages; ++i) mbar_init(&bars[w][i], halves);
    fence_barrier_init();
    tma_prefetch_desc(&kmap);
    tma_prefetch_desc(&vmap);
  }
  if (tid < kStreams * 2) s_start[tid >> 1][tid & 1] = -1;
  pdl_trigger();
  pdl_wait();

  // ---------------------------------------------------------------- the tile list
  {
    const int per = (a.B + kWarps * 32 - 1) / (kWarps * 32);
    const int r0 = min(a.B, tid * per), r1 = min(a.B, r0 + per);
    auto tiles_of = [&](int b) {
      return (long long)Hkv * ((s_first[a.B + b] * G + kRows - 1) / kRows) * ((s_rows[b] + kTile - 1) / kTile);
    };
    long long own = 0;
    for (int b = r0; b < r1; ++b) {
      int first;
      s_first[a.B + b] = q_tokens(a, b, first);
      s_first[b] = first;
      s_rows[b] = rows_of(a, b);
      own += tiles_of(b);
    }
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
  const long long W = prefix[a.B];
  const Split ctas(W, gridDim.x);
  const long long c0 = ctas.begin(blockIdx.x), c1 = ctas.begin(blockIdx.x + 1);
  const long long x0 = c0 + (c1 - c0) * stream / kStreams, x1 = c0 + (c1 - c0) * (stream + 1) / kStreams;
  const Workspace ws = workspace_of(a.workspace, gridDim.x, kStreams, kRows, D);

  auto place_of = [&](long long x) {
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (prefix[mid] <= x) lo = mid;
      else hi = mid;
    }
    Place p;
    p.b = lo;
    p.first = s_first[lo];
    p.qn = s_first[a.B + lo];
    p.n = s_rows[lo];
    const int rts = (p.qn * G + kRows - 1) / kRows;
    p.tiles = (p.n + kTile - 1) / kTile;
    const long long rem = x - prefix[lo];
    const int item = int(quotient(rem, p.tiles));
    p.tile = int(rem - (long long)item * p.tiles);
    p.h = item / rts;
    p.rt = item - p.h * rts;
    return p;
  };

  // ---------------------------------------------------------------- the copies' side (one warp a stream)
  // One lane a page of up to kStep tiles (odd and even tiles of the range have lanes of their own); a
  // page's id is looked up one turn ahead of its copies. The lanes' state lives in shared memory: it is
  // needed once a step, and registers are what limits the number of warps.
  unsigned char* ring = ring_base + stream * S::kRing;
  const bool copies = sub == 0;
  auto look_up = [&](CopyLane& z, long long px, Place pp, int half) {
    z.px = px;
    z.tile = px < x1 ? 1 : 0;
    z.valid = 0;
    if (px < x1) {
      const int block = pp.tile * kTile / P + half;
      if (block * P < pp.n) {
        z.valid = 1;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(&z.page)), "l"(a.table + (long)pp.b * a.width + block)
                     : "memory");
      }
      z.row = pp.tile * kTile % P;
      z.h = pp.h;
    }
    z.pp = pp;
  };
  // K, V and the scales of one page of a tile into a stage; without a page only the arrival
  auto issue = [&](int st, int half, bool valid, int page, int row, int h) {
    uint64_t* bar = &bars[stream][st];
    const int box = min(P, kTile);
    float* sc = meta[stream][st][half];
    if (valid) {
      mbar_expect_tx(bar, 2u * uint32_t(box) * D);
      unsigned char* dst = ring + st * kBytes + half * 16 * D;
      // a page id outside the pool reads as zeros (the tensor map's bounds)
      tma_load_4d(dst, &kmap, bar, row, h, page);
      tma_load_4d(dst + kTile * D, &vmap, bar, row, h, page);
    }
    if (valid && page >= 0 && page < a.c.pages) {
      const long at = (long)page * a.c.scale_page_stride + (long)h * a.c.scale_head_stride;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(sc)), "l"(a.c.k_scale + at) : "memory");
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(sc + 1)), "l"(a.c.v_scale + at) : "memory");
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
    } else {
      if (valid) report_error(a.status, int(StatusCode::kOutOfBounds), 411, page, h);
      sc[0] = sc[1] = 1.f;
      mbar_arrive(bar);
    }
  };
  auto copy = [&](int put_stage, int put_tile, int tiles) {
    if (lane >= kStep * halves) return;
    const int my_tile = lane / halves, my_half = lane % halves;
    const int ahead = my_tile >= put_tile ? my_tile - put_tile : my_tile - put_tile + kStep;
    CopyLane& z = s_copy[stream][lane];
    if (ahead >= tiles || !z.tile) return;
    asm volatile("cp.async.wait_all;" ::: "memory");
    issue(put_stage + ahead >= kStages ? put_stage + ahead - kStages : put_stage + ahead, my_half, z.valid != 0, z.page, z.row, z.h);
    const long long px = z.px + kStep;
    Place pp = z.pp;
    pp.tile += kStep;
    if (pp.tile >= pp.tiles && px < x1) pp = place_of(px);
    look_up(z, px, pp, my_half);
  };
  if (copies && x0 < x1) {
    // the first tiles, every page by a lane of its own, so that their look-ups are one latency
    for (int e = lane; e < kStages * halves; e += 32) {
      const int half = e % halves, st = e / halves;
      if (x0 + st < x1) {
        const Place p = place_of(x0 + st);
        const int block = p.tile * kTile / P + half;
        const bool valid = block * P < p.n;
        issue(st, half, valid, valid ? a.table[(long)p.b * a.width + block] : 0, p.tile * kTile % P, p.h);
      }
    }
    if (lane < kStep * halves) {
      // the lane's first tile of those that follow, in its own place modulo kStep
      const int my_tile = lane / halves;
      const long long px = x0 + kStages + (my_tile + kStep - kStages % kStep) % kStep;
      look_up(s_copy[stream][lane], px, px < x1 ? place_of(px) : Place{}, lane % halves);
    }
  }
  __syncwarp();

  // ---------------------------------------------------------------- rows without an item
  // (no cached rows, or query tokens that belong to no request): o = 0, lse = -inf
  for (int b = blockIdx.x; b < a.B; b += gridDim.x) {
    const int first = s_first[b], qn = s_first[a.B + b];
    const bool some = s_rows[b] > 0;
    const int t0 = b == 0 ? 0 : first, t1 = b + 1 < a.B ? s_first[b + 1] : a.T;
    for (int t = t0; t < min(t1, a.T); ++t) {
      if (some && t >= first) {           // tokens first .. first + qn - 1 have one
        t = max(t, first + qn - 1);
        if (t >= first && t < first + qn) continue;
      }
      uint32_t* o = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.o) + (long)t * a.H * D);
      for (int i = tid; i < a.H * (D / 2); i += kWarps * 32) o[i] = 0u;
      if (a.lse != nullptr)
        for (int h = tid; h < a.H; h += kWarps * 32) a.lse[(long)h * a.T + t] = -INFINITY;
    }
  }

  // ---------------------------------------------------------------- the products' side
  const int j = lane >> 2, c = lane & 3;   // fragment row and column group of the lane
  const int out0 = sub * kOut;             // first piece of O of this warp
  int stage = 0;
  uint32_t phase = 0;                      // of `stage`; a stage before it in the ring is one phase on
  int spent = 0, spent_at = 0, spent_tile = 0;   // team: stages that take copies at the next step
  long long x = x0;
  // A wait that ran out (reported) ends the waiting and the copies, not the loop: the barriers that two
  // warps share stay matched, and the rest of the range is computed on whatever the ring holds. No other
  // report ends it: a bad page id of one request (or a word that an earlier call left set) says nothing
  // about this stream's copies, which land in this CTA's memory and have to be waited for.
  bool alive = true;
  auto stage_at = [&](int i) { return stage + i >= kStages ? stage + i - kStages : stage + i; };
  auto parity_at = [&](int i) { return stage + i >= kStages ? phase ^ 1 : phase; };
  auto await = [&](int q) {
    if (mbar_wait(&bars[stream][stage_at(q)], parity_at(q), nullptr, 0)) return;
    report_error(a.status, int(StatusCode::kMbarTimeout), 412, int(x - x0));
    alive = false;
    // the copies still in flight, together as long again (the ring holds the tiles from x on, without the
    // stages that have not taken a new copy yet)
    const uint64_t t0 = globaltimer_ns();
    for (int i = q + 1; i < kStages - spent && x + i < x1; ++i)
      while (!mbar_try_wait(smem_u32(&bars[stream][stage_at(i)]), parity_at(i)) && globaltimer_ns() - t0 < kPipeTimeoutNs) {}
  };
  while (x < x1) {
    const Place p = place_of(x);
    const int n = p.n, qn = p.qn;
    const int end = int(min((long long)p.tiles, p.tile + (x1 - x)));
    const int r0 = p.rt * kRows, rows = min(qn * G - r0, kRows);   // the item's query rows

    // q as the f16 B operand: lane (j, c) holds row j of each column tile, dims 16 s + 4 c .. + 3 of
    // k step s (the same order in which a lane's K bytes come out of ldmatrix)
    uint32_t qf[kShared ? 1 : NT][kShared ? 1 : kChunks][2];
    uint2* qs = q_frag + stream * kChunks * NT * 32 + lane;
    float m[NT][2], l[NT][2];
    float acc[kOut][NT][4];
    const uint16_t* q_at = reinterpret_cast<const uint16_t*>(a.q) + (long)p.first * a.q_stride + (long)p.h * G * a.q_head_stride + 4 * c;
    auto load_q = [&](int t, float (&v)[kChunks][4]) {
      const int r = t * 8 + j;
      const int qi = (r0 + r) / G, g = (r0 + r) % G;
      const uint16_t* src = q_at + (long)qi * a.q_stride + (long)g * a.q_head_stride;
#pragma unroll
      for (int s = 0; s < kChunks; ++s) {
        const uint2 w = r < rows ? *reinterpret_cast<const uint2*>(src + 16 * s) : make_uint2(0, 0);
        if (a.q_dtype == kBF16) {
          v[s][0] = bf16_lo(w.x); v[s][1] = bf16_hi(w.x); v[s][2] = bf16_lo(w.y); v[s][3] = bf16_hi(w.y);
        } else {
          const float2 lo = half2_floats(w.x), hi = half2_floats(w.y);
          v[s][0] = lo.x; v[s][1] = lo.y; v[s][2] = hi.x; v[s][3] = hi.y;
        }
      }
    };
    // |q| 2^e in [2^14, 2^15) for the item's largest finite element: bf16's 8 bits stay exact in f16
    // down to 2^-31 of it
    float top_q = 0.f;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float v[kChunks][4];
      load_q(t, v);
#pragma unroll
      for (int s = 0; s < kChunks; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) top_q = fmaxf(top_q, fabsf(v[s][i]) < 3.4e38f ? fabsf(v[s][i]) : 0.f);
    }
    top_q = warp_max(top_q);
    const int e2 = top_q > 0.f ? max(-113, min(100, 14 - (((__float_as_int(top_q) >> 23) & 0xff) - 127))) : 0;
    const float factor = a.scale * 1.4426950408889634f * pow2(-e2);   // of the scores, to the log2 domain
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float v[kChunks][4];
      load_q(t, v);
      const float up = pow2(e2);
#pragma unroll
      for (int s = 0; s < kChunks; ++s) {
        const uint32_t lo = pack_half(v[s][0] * up, v[s][1] * up), hi = pack_half(v[s][2] * up, v[s][3] * up);
        if constexpr (kShared) {
          if (sub == t % kTeam) qs[(s * NT + t) * 32] = make_uint2(lo, hi);
        } else {
          qf[t][s][0] = lo;
          qf[t][s][1] = hi;
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        m[t][i] = kNone;
        l[t][i] = 0.f;
      }
#pragma unroll
      for (int s = 0; s < kOut; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[s][t][i] = 0.f;
    }
    if (kShared) team_sync<kTeam>(stream);
    const int qi0 = r0 / G, qi1 = (r0 + rows - 1) / G;    // the item's query tokens
    const int least = n - qn + qi0 + 1;                   // rows that all of them see

    for (int tile = p.tile; tile < end; tile += kStep) {
      const int count = min(kStep, end - tile);           // tiles of this step
#pragma unroll
      for (int q = 0; q < kStep; ++q)
        if (alive && q < count) await(q);
      const int base = tile * kTile;
      const uint32_t ring_at = smem_u32(ring);
      const bool edge = base + kStep * kTile > least || count < kStep;
      // ---- S^T = K Q^T of this warp's 16-token groups: group g is half g % 2 of the step's tile g / 2
      const int g0 = sub * kMt;
      const bool idle = g0 / 2 >= count;                  // its tile is not there in this step
      const int k_stage = stage_at(g0 / 2);
      const uint32_t kbase = ring_at + k_stage * kBytes + (kMt == 2 ? 0 : (g0 & 1) * 16 * D);
      float s[kMt][NT][4];
      float iv[kMt];
      bool dead[kMt];
#pragma unroll
      for (int mt = 0; mt < kMt; ++mt)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[mt][t][i] = 0.f;
#pragma unroll
      for (int k = 0; k < kChunks; k += 2) {
        uint2 qb[2][NT];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            if constexpr (kShared) qb[h][t] = qs[((k + h) * NT + t) * 32];
            else qb[h][t] = make_uint2(qf[t][k + h][0], qf[t][k + h][1]);
          }
#pragma unroll
        for (int mt = 0; mt < kMt; ++mt) {
          uint32_t r[4];
          ldmatrix4(kbase + piece<D>(mt * 16 + (lane & 15), k + (lane >> 4)), r);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t af[4];
            decode4<INT8>(r[2 * h], af[0], af[2]);
            decode4<INT8>(r[2 * h + 1], af[1], af[3]);
#pragma unroll
            for (int t = 0; t < NT; ++t) mma_f16(s[mt][t], af, qb[h][t].x, qb[h][t].y);
          }
        }
      }
      // ---- in the log2 domain, masked; the running maximum
#pragma unroll
      for (int mt = 0; mt < kMt; ++mt) {
        const int half = halves == 2 ? (g0 + mt) & 1 : 0;
        const float ks = meta[stream][k_stage][half][0], vs = meta[stream][k_stage][half][1];
        // a block scaled by 0 holds zeros: its weight counts in l and its p V is 0 whatever p is
        // (the approximate logarithm and quotient are off by a few units of the last place: a page's
        // weights by about 2^-20, in the sum and in O alike, where P's rounding to f16 is 2^-12)
        dead[mt] = vs == 0.f || idle;
        const float lv = dead[mt] ? 0.f : __log2f(vs);
        iv[mt] = dead[mt] ? 1.f : __fdividef(1.f, vs);
        const float2 f = make_float2(factor * ks, factor * ks), lv2 = make_float2(lv, lv);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            const float2 x = __ffma2_rn(make_float2(s[mt][t][i], s[mt][t][i + 1]), f, lv2);
            s[mt][t][i] = x.x;
            s[mt][t][i + 1] = x.y;
          }
      }
      if (edge) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            // rows that query row t * 8 + 2 c + (i & 1) sees (past the item's rows: any)
            const int col = t * 8 + 2 * c + (i & 1);
            const int lim = idle ? 0 : col < rows ? n - qn + (r0 + col) / G + 1 : n;
#pragma unroll
            for (int mt = 0; mt < kMt; ++mt)
              if (base + (g0 + mt) * 16 + j + (i >> 1) * 8 >= lim) s[mt][t][i] = -INFINITY;
          }
      }
      float top[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float v = fmaxf(s[0][t][i], s[0][t][i + 2]);
#pragma unroll
          for (int mt = 1; mt < kMt; ++mt) v = max3f(v, s[mt][t][i], s[mt][t][i + 2]);
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
          top[t][i] = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
        }
      if (kShared) {
        if (j == 0) {
#pragma unroll
          for (int t = 0; t < NT; ++t)
            *reinterpret_cast<float2*>(&s_max[stream][sub][t * 8 + 2 * c]) = make_float2(top[t][0], top[t][1]);
        }
        team_sync<kTeam>(stream);
        // all warps are past the previous step: its stages take the next copies
        if (copies && alive && spent > 0) copy(spent_at, spent_tile, spent);
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int o = 1; o < kTeam; ++o) {
            const float2 v = *reinterpret_cast<const float2*>(&s_max[stream][sub ^ o][t * 8 + 2 * c]);
            top[t][0] = fmaxf(top[t][0], v.x);
            top[t][1] = fmaxf(top[t][1], v.y);
          }
      }
      bool changed = false;
#pragma unroll
      for (int t = 0; t < NT; ++t) changed |= top[t][0] > m[t][0] || top[t][1] > m[t][1];
      if (__any_sync(0xffffffffu, changed)) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          float up[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float now = fmaxf(m[t][i], top[t][i]);
            up[i] = fast_exp2(m[t][i] - now);
            m[t][i] = now;
            l[t][i] *= up[i];
          }
#pragma unroll
          for (int k = 0; k < kOut; ++k)
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              const float2 x = __fmul2_rn(make_float2(acc[k][t][i], acc[k][t][i + 1]), make_float2(up[0], up[1]));
              acc[k][t][i] = x.x;
              acc[k][t][i + 1] = x.y;
            }
        }
      }
      // ---- p, its sum, and P^T as the B operand of a 16-token step
      uint32_t pf[kMt][NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const float2 up = make_float2(kShift - m[t][0], kShift - m[t][1]);
        float2 sum = make_float2(l[t][0], l[t][1]);
#pragma unroll
        for (int mt = 0; mt < kMt; ++mt) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float2 x = __fadd2_rn(make_float2(s[mt][t][2 * i], s[mt][t][2 * i + 1]), up);
            const float2 e = make_float2(fast_exp2(x.x), fast_exp2(x.y));
            sum = __ffma2_rn(e, make_float2(iv[mt], iv[mt]), sum);
            pf[mt][t][i] = transpose8x8(pack_half(e.x, e.y));
          }
        }
        l[t][0] = sum.x;
        l[t][1] = sum.y;
      }
#pragma unroll
      for (int mt = 0; mt < kMt; ++mt) {
        if (dead[mt]) {     // (the same for the warp)
#pragma unroll
          for (int t = 0; t < NT; ++t) pf[mt][t][0] = pf[mt][t][1] = 0u;
        }
        if constexpr (kShared) {
#pragma unroll
          for (int t = 0; t < NT; ++t) s_p[stream][g0 + mt][t][lane] = make_uint2(pf[mt][t][0], pf[mt][t][1]);
        }
      }
      if (kShared) team_sync<kTeam>(stream);
      // ---- O^T += V^T P^T. In a step that ends inside the rows some query token sees, every query
      // token gets a pass of its own with the codes it must not see taken as 0, and only its own
      // columns take the result: whatever a masked place holds (stale bytes behind the end, NaN in a
      // later draft's row), p = 0 cannot cancel it.
      auto values = [&](int q, int seen, bool all) {
        const uint32_t vbase = ring_at + stage_at(q) * kBytes + kTile * D;
#pragma unroll
        for (int mt = 0; mt < 2; ++mt) {
          uint32_t b0[NT], b1[NT];
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            if constexpr (kShared) {
              const uint2 b = s_p[stream][q * 2 + mt][t][lane];
              b0[t] = b.x;
              b1[t] = b.y;
            } else {
              b0[t] = pf[mt][t][0];
              b1[t] = pf[mt][t][1];
            }
          }
          bool mine[NT][2];   // the lane's accumulator columns that take part in this pass
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) mine[t][i] = all || n - qn + (r0 + t * 8 + 2 * c + i) / G + 1 == seen;
          const int tok = base + q * kTile + mt * 16 + 2 * c;
#pragma unroll
          for (int k = 0; k < kOut; k += 2) {
            uint32_t r[4];
            ldmatrix4_trans(vbase + piece<D>(mt * 16 + (lane & 15), out0 + k + (lane >> 4)), r);
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
              for (int t = 0; t < NT; ++t) {
                if (all) {
                  mma_f16(acc[k + h][t], af, b0[t], b1[t]);
                } else {
                  float v[4];
#pragma unroll
                  for (int i = 0; i < 4; ++i) v[i] = acc[k + h][t][i];
                  mma_f16(v, af, b0[t], b1[t]);
#pragma unroll
                  for (int i = 0; i < 4; ++i) acc[k + h][t][i] = mine[t][i & 1] ? v[i] : acc[k + h][t][i];
                }
              }
            }
          }
        }
      };
      if (!edge) {
#pragma unroll
        for (int q = 0; q < kStep; ++q) values(q, 0, true);
      } else {
#pragma unroll 1
        for (int qi = qi0; qi <= qi1; ++qi) {
          const int seen = n - qn + qi + 1;
#pragma unroll 1
          for (int q = 0; q < count; ++q)
            if (seen > base + q * kTile) values(q, seen, false);
        }
      }
      // ---- the stages are free (team: once the other warps are known to be done with them, at the
      // next step's first barrier)
      if (kShared) {
        spent_at = stage;
        // stage i of the prologue took tile i of the range, so a copy's tile modulo kStep follows
        spent_tile = int(x - x0 + kStages) % kStep;
        spent = count;
      }
      x += count;
      if (!kShared) {
        __syncwarp();
        if (alive) copy(stage, 0, 1);
      }
      stage += count;
      if (stage >= kStages) {
        stage -= kStages;
        phase ^= 1;
      }
    }
    // ---------------------------------------------------------------- the item's result
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float v = l[t][i];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        l[t][i] = v + __shfl_xor_sync(0xffffffffu, v, 16);
      }
    if (kShared) {   // each warp has the sums of its own tokens
      team_sync<kTeam>(stream);
      if (j == 0) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
          *reinterpret_cast<float2*>(&s_max[stream][sub][t * 8 + 2 * c]) = make_float2(l[t][0], l[t][1]);
      }
      team_sync<kTeam>(stream);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        l[t][0] = l[t][1] = 0.f;
#pragma unroll
        for (int o = 0; o < kTeam; ++o) {
          const float2 v = *reinterpret_cast<const float2*>(&s_max[stream][o][t * 8 + 2 * c]);
          l[t][0] += v.x;
          l[t][1] += v.y;
        }
      }
      team_sync<kTeam>(stream);
    }
    const bool complete = p.tile == 0 && end == p.tiles;
    const bool last = x >= x1;
    if (complete) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = t * 8 + 2 * c + i;
          if (r < rows) {
            const int qi = (r0 + r) / G, head = p.h * G + (r0 + r) % G;
            const float inv = row_inv(l[t][i]);
            uint32_t* o = reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.o) + ((long)(p.first + qi) * a.H + head) * D);
#pragma unroll
            for (int k = 0; k < kOut; ++k)
              o[(out0 + k) * 8 + j] = pack16(a.q_dtype, acc[k][t][i] * inv, acc[k][t][i + 2] * inv);
            if (j == 0 && sub == 0 && a.lse != nullptr) a.lse[(long)head * a.T + p.first + qi] = row_lse(m[t][i], l[t][i]);
          }
        }
    } else {
      // the range's last piece stays in the stream's ring (free: all its tiles are consumed; the team
      // has just met), a first piece before another item goes to the workspace
      const int slot = last ? 1 : 0;
      float* po = last ? reinterpret_cast<float*>(ring) : ws.head + ((size_t)blockIdx.x * kStreams + stream) * kRows * D;
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = t * 8 + 2 * c + i;
          if (r < rows) {
            float2* o = reinterpret_cast<float2*>(po + (size_t)r * D);
#pragma unroll
            for (int k = 0; k < kOut; ++k) o[(out0 + k) * 8 + j] = make_float2(acc[k][t][i], acc[k][t][i + 2]);
            if (j == 0 && sub == 0) {
              s_ml[stream][slot][r][0] = m[t][i];
              s_ml[stream][slot][r][1] = l[t][i];
            }
          }
        }
      if (lane == 0 && sub == 0) {
        s_start[stream][slot] = x - (end - p.tile) - p.tile;
        s_place[stream][slot] = p;
      }
    }
  }
  __syncthreads();

  // ---------------------------------------------------------------- the CTA's pieces, item by item
  // bit 2 i + k of a mask: piece k of stream i. Every warp finds the items by itself; the threads share
  // (item, row, four dims) so that all pieces of all items are read at once.
  const long long my_start = lane < 2 * kStreams ? s_start[lane >> 1][lane & 1] : -1;
  const uint32_t same = __match_any_sync(0xffffffffu, my_start);
  const uint32_t leaders = __ballot_sync(0xffffffffu, my_start >= 0 && __ffs(same) - 1 == lane);
  const int items = __popc(leaders);
  constexpr int kElems = kRows * (D / 4);     // of an item (a multiple of a warp: a warp's lanes share an item)
  for (int at = tid; at < items * kElems; at += kWarps * 32) {
    const int lead = __fns(leaders, 0, at / kElems + 1);
    const uint32_t mask = __shfl_sync(0xffffffffu, same, lead);
    const long long start = __shfl_sync(0xffffffffu, my_start, lead);
    const Place& p = s_place[lead >> 1][lead & 1];
    const int r = at % kElems / (D / 4), d = at % (D / 4);
    const int r0 = p.rt * kRows, rows = min(p.qn * G - r0, kRows);
    if (r >= rows) continue;
    float top = kNone;
#pragma unroll
    for (int k = 0; k < 2 * kStreams; ++k)
      if (mask >> k & 1) top = fmaxf(top, s_ml[k >> 1][k & 1][r][0]);
    float l = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](int k, const float4 o) {
      const float w = fast_exp2(s_ml[k >> 1][k & 1][r][0] - top);
      l = fmaf(w, s_ml[k >> 1][k & 1][r][1], l);
      v.x = fmaf(w, o.x, v.x);
      v.y = fmaf(w, o.y, v.y);
      v.z = fmaf(w, o.z, v.z);
      v.w = fmaf(w, o.w, v.w);
    };
#pragma unroll
    for (int k = 0; k < 2 * kStreams; ++k)
      if (mask >> k & 1)
        add(k, (k & 1) ? *reinterpret_cast<const float4*>(ring_base + (k >> 1) * S::kRing + ((size_t)r * D + 4 * d) * 4)
                       : *reinterpret_cast<const float4*>(ws.head + (((size_t)blockIdx.x * kStreams + (k >> 1)) * kRows + r) * D + 4 * d));
    if (start >= c0 && start + p.tiles <= c1) {
      const int qi = (r0 + r) / G, head = p.h * G + (r0 + r) % G;
      const float inv = row_inv(l);
      reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.o) + ((long)(p.first + qi) * a.H + head) * D)[d] =
          make_uint2(pack16(a.q_dtype, v.x * inv, v.y * inv), pack16(a.q_dtype, v.z * inv, v.w * inv));
      if (d == 0 && a.lse != nullptr) a.lse[(long)head * a.T + p.first + qi] = row_lse(top, l);
    } else {
      const size_t row = ((size_t)blockIdx.x * 2 + (start < c0 ? 0 : 1)) * kRows + r;
      reinterpret_cast<float4*>(ws.o + row * D)[d] = v;
      if (d == 0) *reinterpret_cast<float2*>(ws.ml + row * 2) = make_float2(top, l);
    }
  }
  if (warp == 0) {
    // the item that starts in this range and goes on past it, if there is one
    const bool open = (leaders >> lane & 1) && my_start >= c0 && my_start + s_place[lane >> 1][lane & 1].tiles > c1;
    const uint32_t who = __ballot_sync(0xffffffffu, open);
    if (open) {
      const Place& p = s_place[lane >> 1][lane & 1];
      const int r0 = p.rt * kRows;
      ws.straddle[blockIdx.x] = Straddle{ctas.part_of(my_start + p.tiles - 1), r0, min(p.qn * G - r0, kRows), p.first, p.h * G, {0, 0, 0}};
    }
    if (who == 0 && lane == 0) ws.straddle[blockIdx.x].last = -1;
  }
}

// One CTA per (CTA of the attention, query row): where that CTA's last item goes on in the next ones,
// their pieces of the row in list order, one warp a piece at a time.
constexpr int kCombineWarps = 8;

template <int D, int NT>
__global__ void __launch_bounds__(kCombineWarps * 32) combine_kernel(AttnArgs a) {
  constexpr int kRows = 8 * NT, kPer = D / 32;
  __shared__ float part[kCombineWarps][D];
  __shared__ float part_ml[kCombineWarps][2];
  pdl_trigger();
  pdl_wait();
  const int cta = blockIdx.x, row = blockIdx.y, grid = gridDim.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Workspace ws = workspace_of(a.workspace, grid, Shape<D, NT>::kStreams, kRows, D);
  const Straddle st = ws.straddle[cta];
  if (row >= st.rows || st.last < 0) return;
  auto at = [&](int w) { return ((size_t)w * 2 + (w == cta ? 1 : 0)) * kRows + row; };
  float acc[kPer], l = 0.f, top = kNone;
#pragma unroll
  for (int i = 0; i < kPer; ++i) acc[i] = 0.f;
#pragma unroll 4
  for (int w = cta + warp; w <= st.last; w += kCombineWarps) {
    const float2 ml = *reinterpret_cast<const float2*>(ws.ml + at(w) * 2);
    const float* o = ws.o + at(w) * D + lane * kPer;
    float2 v[kPer / 2];
#pragma unroll
    for (int i = 0; i < kPer / 2; ++i) v[i] = reinterpret_cast<const float2*>(o)[i];
    const float now = fmaxf(top, ml.x);
    const float keep = fast_exp2(top - now), e = fast_exp2(ml.x - now);
    top = now;
    l = fmaf(e, ml.y, l * keep);
#pragma unroll
    for (int i = 0; i < kPer / 2; ++i) {
      acc[2 * i] = fmaf(e, v[i].x, acc[2 * i] * keep);
      acc[2 * i + 1] = fmaf(e, v[i].y, acc[2 * i + 1] * keep);
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) part[warp][lane * kPer + i] = acc[i];
  if (lane == 0) {
    part_ml[warp][0] = top;
    part_ml[warp][1] = l;
  }
  __syncthreads();
  if (threadIdx.x >= D / 2) return;
  top = kNone;
  l = 0.f;
  float v0 = 0.f, v1 = 0.f;
#pragma unroll
  for (int w = 0; w < kCombineWarps; ++w) top = fmaxf(top, part_ml[w][0]);
#pragma unroll
  for (int w = 0; w < kCombineWarps; ++w) {
    const float e = fast_exp2(part_ml[w][0] - top);
    l = fmaf(e, part_ml[w][1], l);
    v0 = fmaf(e, part[w][2 * threadIdx.x], v0);
    v1 = fmaf(e, part[w][2 * threadIdx.x + 1], v1);
  }
  const int G = a.H / a.c.Hkv, r = st.row0 + row, t = st.first + r / G, head = st.head + r % G;
  const float inv = row_inv(l);
  reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(a.o) + ((long)t * a.H + head) * D)[threadIdx.x] =
      pack16(a.q_dtype, v0 * inv, v1 * inv);
  if (threadIdx.x == 0 && a.lse != nullptr) a.lse[(long)head * a.T + t] = row_lse(top, l);
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

// Column tiles of 8 query rows an item has: the least that hold a request's rows, at most 5. 64 requests
// of up to 32768 rows, 4 KV heads, 128 dims: 7 rows with 1, 2, 3 and 5 tiles 128, 155, 202, 280 us; 14
// rows with 2, 3, 5 167, 210, 290; 21 rows with 3 and 5 220 and 302. 64 dims: 83, 101, 157, 200; 109,
// 165, 208; 171 and 216. There is no shape of 4 tiles: 25 to 32 rows take that of 5.
int column_tiles(const AttnArgs& a) {
  const long rows = (long)a.max_q * (a.H / a.c.Hkv);
  return rows <= 8 ? 1 : rows <= 16 ? 2 : rows <= 24 ? 3 : 5;
}

template <int D, int NT, bool INT8>
cudaError_t launch_attn(const AttnArgs& a, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t s) {
  using S = Shape<D, NT>;
  const size_t ring = 1024 + size_t(S::kStreams) * S::kRing + S::kQBytes;
  constexpr size_t kPerRequest = sizeof(long long) + 3 * sizeof(int);
  const size_t smem = ring + size_t(a.B + 1) * kPerRequest;
  auto kernel = attn_kernel<D, NT, INT8>;
  cudaError_t e = once_per_device_kernel(reinterpret_cast<const void*>(kernel), [&] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(ring + (kAttnMaxRows + 1) * kPerRequest));
  });
  if (e != cudaSuccess) return e;
  e = launch_pdl(kernel, dim3(unsigned(a.num_sms)), dim3(S::kThreads), smem, s, km, vm, a);
  if (e != cudaSuccess) return e;
  // the rows that an item can have whatever max_q says (a loop over further rows in each CTA: 0.4 us more)
  const long rows = std::min<long>((a.cu == nullptr ? 1l : (long)a.T) * (a.H / a.c.Hkv), S::kRows);
  return launch_pdl(combine_kernel<D, NT>, dim3(unsigned(a.num_sms), unsigned(rows)), dim3(kCombineWarps * 32), 0, s, a);
}

template <int D, int NT>
cudaError_t attn_code(const AttnArgs& a, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t s) {
  return a.c.code == kInt8 ? launch_attn<D, NT, true>(a, km, vm, s) : launch_attn<D, NT, false>(a, km, vm, s);
}

template <int D>
cudaError_t attn_rows(const AttnArgs& a, const CUtensorMap& km, const CUtensorMap& vm, cudaStream_t s) {
  switch (column_tiles(a)) {
    case 1: return attn_code<D, 1>(a, km, vm, s);
    case 2: return attn_code<D, 2>(a, km, vm, s);
    case 3: return attn_code<D, 3>(a, km, vm, s);
    default: return attn_code<D, 5>(a, km, vm, s);
  }
}

}  // namespace

size_t attention_workspace(const AttnArgs& a) {
  const int nt = column_tiles(a);
  auto bytes = [&](auto shape) { return workspace_of(nullptr, a.num_sms, shape.kStreams, shape.kRows, a.c.D).bytes; };
  if (a.c.D == 64)
    return nt == 1 ? bytes(Shape<64, 1>{}) : nt == 2 ? bytes(Shape<64, 2>{}) : nt == 3 ? bytes(Shape<64, 3>{}) : bytes(Shape<64, 5>{});
  return nt == 1 ? bytes(Shape<128, 1>{}) : nt == 2 ? bytes(Shape<128, 2>{}) : nt == 3 ? bytes(Shape<128, 3>{}) : bytes(Shape<128, 5>{});
}

const char* attention(const AttnArgs& a, cudaStream_t s) {
  const Cache& c = a.c;
  if (c.D != 64 && c.D != 128) return "attention_kv8: head_dim must be 64 or 128";
  if (c.P != 16 && c.P != 32 && c.P != 64 && c.P != 128) return "attention_kv8: page must be 16, 32, 64 or 128 tokens";
  if (a.H < 1 || c.Hkv < 1 || a.H % c.Hkv) return "attention_kv8: heads must be a multiple of the KV heads";
  if (a.B > kAttnMaxRows) return "attention_kv8: at most 1024 requests";
  if ((long)a.T * a.H > 0x7fffffc0l || (long)a.max_q * a.H > 0x3fffffffl || (long)a.width * c.P > 0x7fffffc0l)
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
  const cudaError_t e = c.D == 64 ? attn_rows<64>(a, km, vm, s) : attn_rows<128>(a, km, vm, s);
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace kv8
}  // namespace hcp
