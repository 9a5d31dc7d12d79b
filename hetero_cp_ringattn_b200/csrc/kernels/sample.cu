// Batched sampling with temperature, top-k, top-p and min-p from given uniform numbers.
//
// For a row of logits l with maximum L (NaN counts as -inf) and temperature T > 0:
//   d_i = (L - l_i) / T                       distance from the maximum, >= 0
//   w_i = floor(2^31 exp(-d_i))               fixed-point weight, an integer
// Tokens are ordered by (d, index). Top-k keeps the first k; top-p keeps, of those, the tokens
// whose exclusive cumulative weight lies below max(1, floor(top_p * their total)); min-p keeps
// w_i >= floor(2^31 min_p). With S the kept total, the token is the first one in vocabulary order
// whose inclusive cumulative kept weight exceeds floor(u S) (top_p and u in 24 bits). T <= 0: the
// lowest index of the maximum. A row without a finite or +inf logit gives -1.
//
// The weights come from a fixed sequence of IEEE operations (each rounded by itself) and everything
// after them is integer arithmetic, so sums do not depend on the order in which they are taken: the
// same token on the CPU, on the GPU and however a row is split. Weights below 2^-31 of the largest
// are 0; u has 24 bits and cannot reach them.
//
// One cluster per row: each CTA holds a contiguous slice of the row in shared memory, so the logits
// are read from memory once. A histogram over d (bins of 1/32; counts for top-k, counts and weight
// sums for top-p) gives the bin where the cut falls; the tokens up to it, usually a few dozen, are
// sent to one CTA, sorted and finished there. A top-k of up to 256 gets its bin from the threads'
// maxima instead (129 rows of 151936 tokens, k = 40: 70 us; with a count of every token 83). More than
// 512 of them (a large k, a flat row, ties) take the general way: histograms of the crossing bin until
// it is small, or the exact tie, then one pass over the kept tokens.
//
// Bound: the phases of a row, one after another: its load, the cluster's maximum, the work on its
// tokens, further cluster barriers. One row is that chain; of many rows two CTAs an SM overlap two chains,
// which fills neither pipe (issue slots 33%, DRAM 9%, as many stalls on barriers as on fixed latencies).
// The weight's polynomial runs on packed pairs. Measured on B200, float32 logits: one row of
// 128256 tokens 20 us; 129 rows of 151936 (78 MB, 12 us of reading) 102 us with mixed settings, greedy
// alone 32, temperature alone 62, top-k 40 70, top-k 1000 119, top-p 0.9 over random logits (the
// general way) 183. One CTA a row that reads the row again in every pass instead of holding it: 289.
#include <cooperative_groups.h>

#include <cuda_bf16.h>

#include <algorithm>

#include "common.cuh"
#include "launch.h"
#include "sample.h"

namespace hcp {
namespace sampling {

using namespace hcp::dev;
namespace cg = cooperative_groups;

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 512;        // two CTAs an SM: one row's barriers hide behind another's work
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 1024;
constexpr float kPerUnit = 32.f;      // bins per unit of d
constexpr int kList = kThreads;     // tokens that are ordered directly (one a thread)
constexpr int kMaxCluster = 16;     // 16 is the hardware's limit (above 8: opt-in)
constexpr int kMaxSlice = 45056;    // floats of a row in one CTA's shared memory
constexpr int kPairSlice = 20480;   // and where two CTAs share an SM
constexpr u64 kAll = ~0ull;

// Operations on logits and distances: no contraction, no flush of subnormals, whatever the flags.
__device__ __forceinline__ float sub_rn(float a, float b) {
  float r;
  asm("sub.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float div_rn(float a, float b) {
  float r;
  asm("div.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

__device__ __forceinline__ float max_rn(float a, float b) {   // (a NaN operand: the other one)
  float r;
  asm("max.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float min_rn(float a, float b) {
  float r;
  asm("min.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ bool equal(float a, float b) {
  uint32_t r;
  asm("{\n\t.reg .pred p;\n\tsetp.eq.f32 p, %1, %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r) : "f"(a), "f"(b));
  return r != 0;
}
__device__ __forceinline__ float warp_max_rn(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = max_rn(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// floor(2^31 exp(-d)) for 0 <= d <= 64: y = d log2(e), n = round(y), 2^(n - y) on [-1/2, 1/2] by the
// Taylor series of 2^g to degree 7 (remainder below 1e-8), then a shift by n. Adding and subtracting
// 1.5 * 2^23 rounds y to the nearest integer (ties to even) and leaves it in the sum's low bits.
__device__ __forceinline__ uint2 weight2(float d0, float d1) {
  auto pair = [](float x) { return make_float2(x, x); };
  const float2 y = __fmul2_rn(make_float2(d0, d1), pair(0x1.715476p+0f));
  const float2 t = __fadd2_rn(y, pair(12582912.f));
  const float2 n = __fadd2_rn(t, pair(-12582912.f));
  const float2 g = __fadd2_rn(n, make_float2(-y.x, -y.y));
  float2 w = __fadd2_rn(__fmul2_rn(pair(0x1.ffcbfcp-17f), g), pair(0x1.430912p-13f));
  w = __fadd2_rn(__fmul2_rn(w, g), pair(0x1.5d87fep-10f));
  w = __fadd2_rn(__fmul2_rn(w, g), pair(0x1.3b2ab6p-7f));
  w = __fadd2_rn(__fmul2_rn(w, g), pair(0x1.c6b08ep-5f));
  w = __fadd2_rn(__fmul2_rn(w, g), pair(0x1.ebfbep-3f));
  w = __fadd2_rn(__fmul2_rn(w, g), pair(0x1.62e43p-1f));
  w = __fadd2_rn(__fmul2_rn(w, g), pair(1.0f));
  // w in (0.7, 1.42): 24 significant bits at 2^-23 or 2^-24 (one place further down)
  auto fixed = [](float v, float sum) {
    const uint32_t b = __float_as_uint(v);
    const uint32_t sh = (__float_as_uint(sum) & 0x7f) + (127 - (b >> 23));
    uint32_t r;
    asm("shr.u32 %0, %1, %2;" : "=r"(r) : "r"((b << 8) | 0x80000000u), "r"(sh));   // (more than 31: 0)
    return r;
  };
  return make_uint2(fixed(w.x, t.x), fixed(w.y, t.y));
}
__device__ __forceinline__ uint32_t weight(float d) { return weight2(d, d).x; }

// floor(32 d), at most kBins - 1 (d <= 64: adding 2^23 towards zero leaves the floor in the low bits).
__device__ __forceinline__ int bin_of(float d) {
  return min(int(__float_as_uint(__fadd_rz(d * kPerUnit, 8388608.f)) & 0x7fffff), kBins - 1);
}

// floor(total * x) for x in [0, 1], x held in 24 bits (total < 2^54).
__device__ __forceinline__ u64 share(u64 total, float x) {
  const float f = x * 16777216.f;
  const u64 q = f > 0.f ? min(u64(f), u64(1) << 24) : 0;
  return (total >> 24) * q + (((total & 0xffffffull) * q) >> 24);
}

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__device__ __forceinline__ u64 warp_scan64(u64 v, int lane) {   // inclusive
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const u64 up = __shfl_up_sync(0xffffffffu, v, d);
    if (lane >= d) v += up;
  }
  return v;
}

struct __align__(16) Shared {
  // this CTA's histogram: x: count in the low 16 bits, carries of y in the high ones; y: weights
  // modulo 2^32 (a slice has at most 45056 tokens of at most 2^31, so both halves hold)
  uint2 hist[kBins];
  u64 slot_c[kMaxCluster], slot_w[kMaxCluster];  // totals of every CTA's segment of bins
  u64 list[kList];                               // this CTA's gathered tokens, (key, index)
  u64 all[kList];                                // the cluster's
  u64 warp_a[kWarps], warp_b[kWarps];
  u64 slot[2][kMaxCluster];                      // one value of every CTA, pushed by it
  float fslot[kMaxCluster];
  int list_n, sent;
  u64 found;                                     // results one thread hands to the block
  u64 found_cnt, found_w, found_in_cnt;
  int found_bin;
};

// Ascending bitonic sort of one u64 a thread, `size` a power of two of threads (the rest idle along).
// Exchanges within a warp are shuffles, wider ones go through `buf`.
__device__ __forceinline__ u64 sort64(u64 v, int size, u64* buf, int tid) {
  for (int k = 2; k <= size; k <<= 1) {
    for (int j = k >> 1; j > 0; j >>= 1) {
      u64 o;
      if (j >= 32) {
        __syncthreads();
        if (tid < size) buf[tid] = v;
        __syncthreads();
        o = tid < size ? buf[tid ^ j] : 0;
      } else {
        o = __shfl_xor_sync(0xffffffffu, v, j);
      }
      const bool low = (tid & j) == 0, up = (tid & k) == 0;
      if (tid < size) v = (low == up) ? (o < v ? o : v) : (o > v ? o : v);
    }
  }
  return v;
}

template <bool BF16>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(SampleArgs a, int slice) {
  extern __shared__ __align__(16) unsigned char raw[];
  Shared& S = *reinterpret_cast<Shared*>(raw);
  cg::cluster_group cluster = cg::this_cluster();
  const int C = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  // the cluster's sums of this CTA's segment of bins, and its slice of the row
  u64* seg_w = reinterpret_cast<u64*>(raw + sizeof(Shared));
  uint32_t* seg_c = reinterpret_cast<uint32_t*>(seg_w + kBins / C);
  float* x = reinterpret_cast<float*>(seg_c + kBins / C);
  const int b = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  cluster.barrier_arrive();   // waited for before the first access to another CTA's shared memory
  pdl_trigger();
  pdl_wait();

  // ---------------------------------------------------------------- the slice and the maximum
  const int lo = min(a.V, rank * slice), n = min(a.V, lo + slice) - lo;
  const int seg = (n + kWarps * 32 - 1) / (kWarps * 32) * 32;   // one warp's run of the slice
  const int s0 = min(n, warp * seg), s1 = min(n, s0 + seg);
  const float ninf = __int_as_float(0xff800000);
  float top = ninf;
  {
    const int esize = BF16 ? 2 : 4, vec = 16 / esize;
    const char* src = reinterpret_cast<const char*>(a.logits) + ((long)b * a.row_stride + lo) * esize;
    const bool aligned = reinterpret_cast<uintptr_t>(src) % 16 == 0;
    const int nv = aligned ? n / vec : 0;
    float4* x4 = reinterpret_cast<float4*>(x);
#pragma unroll 4
    for (int i = tid; i < nv; i += kThreads) {   // (fmaxf passes NaN over)
      const uint4 v = ld_nc_v4(src + (long)i * 16);
      if (BF16) {
        const float4 p = make_float4(bf16_lo(v.x), bf16_hi(v.x), bf16_lo(v.y), bf16_hi(v.y));
        const float4 q = make_float4(bf16_lo(v.z), bf16_hi(v.z), bf16_lo(v.w), bf16_hi(v.w));
        x4[2 * i] = p;
        x4[2 * i + 1] = q;
        top = max_rn(top, max_rn(max_rn(max_rn(p.x, p.y), max_rn(p.z, p.w)), max_rn(max_rn(q.x, q.y), max_rn(q.z, q.w))));
      } else {
        const float4 p = make_float4(__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w));
        x4[i] = p;
        top = max_rn(top, max_rn(max_rn(p.x, p.y), max_rn(p.z, p.w)));
      }
    }
    for (int i = nv * vec + tid; i < n; i += kThreads) {
      const float f = BF16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(src)[i])
                           : reinterpret_cast<const float*>(src)[i];
      x[i] = f;
      top = max_rn(top, f);
    }
  }
  const float own = top;
  const float temp = a.temperature.ptr ? a.temperature.ptr[b] : a.temperature.value;
  const int top_k = a.top_k.ptr ? a.top_k.ptr[b] : a.top_k.value;
  const float top_p = a.top_p.ptr ? a.top_p.ptr[b] : a.top_p.value;
  const float min_p = a.min_p.ptr ? a.min_p.ptr[b] : a.min_p.value;
  const bool greedy = !(temp > 0.f);
  const bool use_k = !greedy && top_k > 0 && top_k < a.V;
  const bool use_p = !greedy && top_p > 0.f && top_p < 1.f;
  auto clear = [&] {
    for (int i = tid; i < kBins; i += kThreads) S.hist[i] = make_uint2(0, 0);
  };
  if (use_k || use_p) clear();
  if (tid == 0) S.list_n = S.sent = 0;
  top = warp_max_rn(top);
  float* wf = reinterpret_cast<float*>(S.warp_a);
  if (lane == 0) wf[warp] = top;
  cluster.barrier_wait();
  __syncthreads();
  top = warp_max_rn(wf[lane % kWarps]);
  if (tid < C) *cluster.map_shared_rank(&S.fslot[rank], tid) = top;
  cluster.sync();
  top = S.fslot[0];
  for (int i = 1; i < C; ++i) top = max_rn(top, S.fslot[i]);

  if (top == ninf) {   // nothing to draw (the whole cluster agrees)
    if (rank == 0 && tid == 0) a.token[b] = -1;
    return;
  }
  if (greedy) {
    uint32_t best = 0xffffffffu;
    for (int i = s0 + lane; i < s1; i += 32)
      if (equal(x[i], top)) best = min(best, uint32_t(lo + i));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = min(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) S.warp_b[warp] = best;
    __syncthreads();
    if (tid == 0) {
      u64 m = S.warp_b[0];
      for (int i = 1; i < kWarps; ++i) m = min(m, S.warp_b[i]);
      *cluster.map_shared_rank(&S.slot[0][rank], 0) = m;
    }
    cluster.sync();
    if (rank == 0 && tid == 0) {
      u64 m = S.slot[0][0];
      for (int i = 1; i < C; ++i) m = min(m, S.slot[0][i]);
      a.token[b] = (long long)m;
    }
    return;
  }

  auto add_to_bin = [&](int bin, uint32_t w) {
    uint32_t one = 1;
    if (w) {
      const uint32_t was = atomicAdd(&S.hist[bin].y, w);
      if (was + w < was) one += 0x10000u;     // the carry of a 64-bit sum
    }
    atomicAdd(&S.hist[bin].x, one);
  };
  const bool filter = use_k || use_p;
  const uint32_t min_w = min_p > 0.f ? uint32_t(fminf(min_p, 1.f) * 2147483648.f) : 0u;
  // (top - l) / T, correctly rounded: by the reciprocal and one correction of the quotient (Markstein
  // 1990: with r = RN(1 / T), q = RN(x r) and e = x - q T exact in a fused multiply-add, RN(q + e r)
  // is RN(x / T)) where no step can leave the normal range (a finite top of at least 2^-30 keeps every
  // nonzero difference above 2^-60); else by division. min(NaN, 64) = 64: NaN logits and
  // infinite distances end beyond every weight.
  const float inv_t = div_rn(1.f, temp);
  const bool by_inverse = temp >= 0x1p-60f && temp <= 0x1p60f && fabsf(top) >= 0x1p-30f && fabsf(top) < 3.4e38f;
  auto distance2 = [&](float2 l) {
    if (by_inverse) {
      const float2 v = __fadd2_rn(make_float2(top, top), make_float2(-l.x, -l.y));
      const float2 r = make_float2(inv_t, inv_t), q = __fmul2_rn(v, r);
      const float2 e = __ffma2_rn(make_float2(-q.x, -q.y), make_float2(temp, temp), v);
      const float2 d = __ffma2_rn(e, r, q);
      return make_float2(min_rn(d.x, 64.f), min_rn(d.y, 64.f));
    }
    auto one = [&](float v) { return equal(v, top) ? 0.f : min_rn(div_rn(sub_rn(top, v), temp), 64.f); };
    return make_float2(one(l.x), one(l.y));
  };
  auto publish = [&] { cluster.sync(); };
  // this warp's, the lower CTAs' and the cluster's sum of `v`, one value a lane, through slot[which]
  auto sum_over = [&](u64 v, int which, u64& mine, u64& below, u64& total) {
    mine = warp_sum64(v);
    if (lane == 0) S.warp_a[warp] = mine;
    __syncthreads();
    const u64 w = lane < kWarps ? S.warp_a[lane] : 0;
    if (warp == 0) {
      const u64 t = warp_sum64(w);
      if (lane < C) *cluster.map_shared_rank(&S.slot[which][rank], lane) = t;
    }
    publish();
    below = warp_sum64(lane < warp ? w : 0);   // the lower warps of this CTA
    total = 0;
    for (int r = 0; r < C; ++r) {
      if (r < rank) below += S.slot[which][r];
      total += S.slot[which][r];
    }
  };
  // The first token in vocabulary order whose inclusive cumulative kept weight exceeds the target. The
  // warp whose run holds it looks at 1024 tokens at a time: each lane sums 32 neighbours (starting at
  // its own offset among them, for the banks), then the lanes share the 32 of the lane that reaches it.
  auto draw = [&](auto kept, u64 mine, u64 below, u64 total) {
    const u64 target = share(total, fminf(a.u[b], 0.99999994f));
    if (target < below || target >= below + mine) return;
    for (int base = s0; base < s1; base += 1024) {
      u64 v = 0;
      for (int j = 0; j < 32; ++j) {
        const int i = base + 32 * lane + ((j + lane) & 31);
        v += i < s1 ? kept(i) : 0u;
      }
      const u64 inc = warp_scan64(v, lane);
      const uint32_t hit = __ballot_sync(0xffffffffu, below + inc > target);
      if (hit) {
        const int l = __ffs(hit) - 1;
        below += __shfl_sync(0xffffffffu, inc - v, l);
        const int i = base + 32 * l + lane;
        const u64 one = warp_scan64(i < s1 ? kept(i) : 0u, lane);
        const uint32_t at = __ballot_sync(0xffffffffu, below + one > target);
        if (lane == __ffs(at) - 1) a.token[b] = lo + i;
        break;
      }
      below += __shfl_sync(0xffffffffu, inc, 31);
    }
  };
  // ---------------------------------------------------------------- the bin of the cut
  // The bin where the cluster's count (or weight) reaches `target` (or top_p of the weight in all the
  // bins, for target 0, which it returns). Every CTA sums
  // one segment of the bins (weights only with `sums`) over the cluster (reading all of every histogram in every CTA would take
  // C times the distributed-memory traffic, which is what this costs), the segments' totals say whose
  // segment the crossing is in, and that CTA tells the others.
  auto find_bin = [&](bool by_weight, u64 target, u64 base_cnt, u64 base_w, bool sums = true) {
    const int per = kBins / C;                 // C is a power of two of at most 16
    const int from = tid % C;
#pragma unroll
    for (int p = tid; p < kBins; p += kThreads) {
      const int i = p / C;
      const uint2 h = *cluster.map_shared_rank(&S.hist[rank * per + i], from);
      uint32_t c = h.x & 0xffffu;
      for (int o = C >> 1; o > 0; o >>= 1) c += __shfl_xor_sync(0xffffffffu, c, o);
      if (from == 0) seg_c[i] = c;
      if (sums) {
        u64 w = (u64(h.x >> 16) << 32) + h.y;
        for (int o = C >> 1; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
        if (from == 0) seg_w[i] = w;
      }
    }
    __syncthreads();
    const int mine_n = (per + kThreads - 1) / kThreads;    // bins a thread looks at
    u64 tc = 0, tw = 0;
    for (int j = 0; j < mine_n; ++j) {
      const int i = tid * mine_n + j;
      if (i < per) {
        tc += seg_c[i];
        if (sums) tw += seg_w[i];
      }
    }
    const u64 ic = warp_scan64(tc, lane), iw = sums ? warp_scan64(tw, lane) : 0;
    if (lane == 31) {
      S.warp_a[warp] = ic;
      S.warp_b[warp] = iw;
    }
    if (tid == 0) S.found_bin = -1;
    __syncthreads();
    const u64 oc = lane < kWarps ? S.warp_a[lane] : 0, ow = lane < kWarps ? S.warp_b[lane] : 0;
    if (warp == 0) {
      const u64 t0 = warp_sum64(oc), t1 = sums ? warp_sum64(ow) : 0;
      if (lane < C) {
        *cluster.map_shared_rank(&S.slot_c[rank], lane) = t0;
        *cluster.map_shared_rank(&S.slot_w[rank], lane) = t1;
      }
    }
    publish();
    u64 ec = base_cnt + ic - tc + warp_sum64(lane < warp ? oc : 0);
    u64 ew = base_w + (sums ? iw - tw + warp_sum64(lane < warp ? ow : 0) : 0);
    u64 all_w = 0;
    for (int r = 0; r < C; ++r) {
      if (r < rank) {
        ec += S.slot_c[r];
        ew += S.slot_w[r];
      }
      all_w += S.slot_w[r];
    }
    if (target == 0) target = max(share(all_w, top_p), u64(1));
    for (int j = 0; j < mine_n; ++j) {
      const int i = tid * mine_n + j;
      if (i >= per) break;
      const u64 c = seg_c[i], w = sums ? seg_w[i] : 0;
      const u64 before = by_weight ? ew : ec, in = by_weight ? w : c;
      if (before < target && before + in >= target) {
        for (int r = 0; r < C; ++r) {
          Shared* o = cluster.map_shared_rank(&S, r);
          o->found_bin = rank * per + i;
          o->found_cnt = ec;
          o->found_w = ew;
          o->found_in_cnt = c;
        }
      }
      ec += c;
      ew += w;
    }
    publish();
    return target;
  };
  auto fill_all = [&] {
    publish();                 // every CTA has read the histogram in place
    clear();
    __syncthreads();
    for (int i = s0 + lane; i < s1; i += 32) add_to_bin(bin_of(x[i]), weight(x[i]));
    publish();
  };
  // Rank 0: the gathered tokens ordered, cut, and the draw among them.
  auto finish = [&](int n_all, bool by_k, u64 limit) {
    int size = 32;
    while (size < n_all) size <<= 1;
    u64 v = tid < n_all ? S.all[tid] : kAll;
    v = sort64(v, size, S.list, tid);
    const bool here = tid < n_all;
    const uint32_t w = here ? weight(__uint_as_float(uint32_t(v >> 32))) : 0u;
    auto scan = [&](u64 val, u64& inc, u64& all) {   // inclusive over the block
      inc = warp_scan64(val, lane);
      __syncthreads();
      if (lane == 31) S.warp_a[warp] = inc;
      __syncthreads();
      const u64 o = lane < kWarps ? S.warp_a[lane] : 0;
      inc += warp_sum64(lane < warp ? o : 0);
      all = warp_sum64(o);
    };
    u64 inc, all;
    bool keep = here && (!by_k || tid < top_k);
    scan(keep ? w : 0u, inc, all);
    if (use_p) keep = keep && inc - w < (by_k ? max(share(all, top_p), u64(1)) : limit);
    keep = keep && w >= min_w;
    // kept tokens in vocabulary order, (index, weight)
    v = sort64(keep ? (u64(uint32_t(v)) << 32) | w : kAll, size, S.list, tid);
    keep = v != kAll;
    scan(keep ? uint32_t(v) : 0u, inc, all);
    const u64 target = share(all, fminf(a.u[b], 0.99999994f));
    if (keep && inc > target && inc - uint32_t(v) <= target) a.token[b] = (long long)(v >> 32);
  };

  // ---------------------------------------------------------------- top-k by the threads' maxima
  // The k-th largest of the threads' maxima bounds the k-th largest token from below, so the bin where
  // their counts reach k holds the cut or lies behind it: one count a thread instead of one a token, and
  // only the tokens up to that bin need a distance. Their number is not known ahead (each CTA sends
  // at most one more than fit); too many of them, or a k the threads cannot bound, take the way below.
  if (use_k && top_k <= kList / 2) {
    atomicAdd(&S.hist[bin_of(distance2(make_float2(own, own)).x)].x, 1u);
    publish();
    find_bin(false, u64(top_k), 0, 0, false);
    const int bin = S.found_bin;
    bool done = false;
    if (bin >= 0 && bin < kBins - 1) {
      const float end = float(bin + 1) * (1.f / kPerUnit);
      // a logit below this is farther than `end`, whatever rounds (no bound outside the normal range)
      const float reach = end * temp;
      const float least = by_inverse ? top - reach * 1.000001f - (fabsf(top) + reach) * 1e-6f : ninf;
      Shared* to = cluster.map_shared_rank(&S, 0);
      auto send = [&](float l, int i) {
        if (l < least) return;
        const float d = distance2(make_float2(l, l)).x;
        if (!(d < end) || atomicAdd(&S.sent, 1) > kList) return;
        const int at = atomicAdd(&to->list_n, 1);
        if (at < kList) to->all[at] = (u64(__float_as_uint(d)) << 32) | uint32_t(lo + i);
      };
      for (int i = s0 + 2 * lane; i < s1; i += 64) {
        const float2 l = *reinterpret_cast<const float2*>(x + i);
        send(l.x, i);
        if (i + 1 < s1) send(l.y, i + 1);
      }
      publish();
      const int n_all = to->list_n;
      cluster.barrier_arrive();          // rank 0's count has been read
      done = n_all <= kList;
      if (done && rank == 0) finish(n_all, true, 0);
      cluster.barrier_wait();
    }
    if (done) return;
    if (tid == 0) S.list_n = 0;
    clear();
    __syncthreads();
  }

  // ---------------------------------------------------------------- distances, totals, histogram
  u64 sum = 0;                // without a filter: of the kept weights
  for (int i = s0 + 2 * lane; i < s1; i += 64) {
    // (slices start 8 elements aligned and a pair past the end stays inside the slice's memory)
    float2 d = distance2(*reinterpret_cast<const float2*>(x + i));
    const bool two = i + 1 < s1;
    if (!two) d.y = 64.f;
    *reinterpret_cast<float2*>(x + i) = d;
    if (use_k) {              // counts alone
      atomicAdd(&S.hist[bin_of(d.x)].x, 1u);
      if (two) atomicAdd(&S.hist[bin_of(d.y)].x, 1u);
      continue;
    }
    const uint2 w = weight2(d.x, d.y);
    if (use_p) {
      add_to_bin(bin_of(d.x), w.x);
      if (two) add_to_bin(bin_of(d.y), w.y);
    } else {
      sum += u64(w.x >= min_w ? w.x : 0u) + (w.y >= min_w ? w.y : 0u);
    }
  }
  u64 mine, below, total;
  if (!filter) {
    sum_over(sum, 0, mine, below, total);
    draw([&](int i) {
      const uint32_t w = weight(x[i]);
      return w >= min_w ? w : 0u;
    }, mine, below, total);
    return;
  }

  bool by_k = use_k;
  publish();                   // the histograms are complete
  u64 limit = find_bin(!by_k, by_k ? u64(top_k) : 0, 0, 0, !by_k);
  if (by_k && (S.found_bin < 0 || S.found_bin == kBins - 1)) {
    // the last bin holds only weights of 0: a top-k cut inside it leaves the draw as it is
    by_k = false;
    if (use_p) {
      fill_all();
      limit = find_bin(true, 0, 0, 0);
    }
  }
  const bool cut_somewhere = by_k || use_p;
  int bin = S.found_bin;
  u64 bin_cnt = S.found_cnt, bin_w = S.found_w, bin_in = S.found_in_cnt;
  // the first level's bin b holds the keys of d in [b / 32, (b + 1) / 32)
  auto first_lo = [](int i) { return __float_as_uint(float(i) * (1.f / kPerUnit)); };

  // ---------------------------------------------------------------- few tokens up to it: one CTA's work
  if (cut_somewhere && bin >= 0 && bin_cnt + bin_in <= kList) {
    const float end = float(bin + 1) * (1.f / kPerUnit);
    Shared* to = cluster.map_shared_rank(&S, 0);
    auto send = [&](float d, int i) {
      if (d < end) to->all[atomicAdd(&to->list_n, 1)] = (u64(__float_as_uint(d)) << 32) | uint32_t(lo + i);
    };
    for (int i = s0 + 2 * lane; i < s1; i += 64) {
      const float2 d = *reinterpret_cast<const float2*>(x + i);   // (past the end: 64)
      send(d.x, i);
      send(d.y, i + 1);
    }
    publish();                 // the last access to another CTA's shared memory is behind it
    if (rank == 0) finish(S.list_n, by_k, limit);
    return;
  }

  // ---------------------------------------------------------------- the general way
  // The (key, index) of the last kept token, by key ranges: tokens in [key_lo, key_hi], `in_cnt` of
  // them, `base` ahead of them. kept_w: the kept prefix's weight.
  u64 cut = kAll;
  const uint32_t* xkey = reinterpret_cast<const uint32_t*>(x);
  bool dirty = false;          // the first level's histogram has been overwritten
  auto order_list = [&](uint32_t key_lo, uint32_t key_hi, bool by_weight, u64 target, u64 base_cnt, u64 base_w, u64& kept_w) {
    for (int i = s0 + lane; i < s1; i += 32) {
      const uint32_t key = xkey[i];
      if (key >= key_lo && key <= key_hi) {
        const int at = atomicAdd(&S.list_n, 1);
        if (at < kList) S.list[at] = (u64(key) << 32) | uint32_t(lo + i);
      }
    }
    publish();
    // lane r looks at CTA r's list; thread t takes token t of the lists laid end to end
    int len = lane < C ? min(cluster.map_shared_rank(&S, lane)->list_n, kList) : 0, n_all = 0;
    u64 v = kAll;
    for (int r = 0; r < C; ++r) {
      const int m = __shfl_sync(0xffffffffu, len, r);
      if (tid >= n_all && tid < n_all + m) v = cluster.map_shared_rank(&S, r)->list[tid - n_all];
      n_all += m;
    }
    publish();                 // every CTA has read the lists
    if (tid == 0) S.list_n = 0;
    int size = 32;
    while (size < n_all) size <<= 1;
    v = sort64(v, size, S.list, tid);
    const uint32_t w = tid < n_all ? weight(__uint_as_float(uint32_t(v >> 32))) : 0u;
    u64 inc = warp_scan64(w, lane);
    __syncthreads();
    if (lane == 31) S.warp_a[warp] = inc;
    if (tid == 0) {
      S.found = kAll;
      S.found_w = 0;
    }
    __syncthreads();
    inc += base_w + warp_sum64(lane < warp ? S.warp_a[lane] : 0);
    const u64 before = by_weight ? inc - w : base_cnt + tid, in = by_weight ? w : 1;
    if (tid < n_all && before < target && before + in >= target) {
      S.found = v;
      S.found_w = inc;
    }
    __syncthreads();
    kept_w = S.found_w;
    const u64 id = S.found;
    __syncthreads();
    return id;
  };
  auto refine = [&](uint32_t key_lo, uint32_t key_hi, bool by_weight, u64 target, u64 base_cnt, u64 base_w, u64 in_cnt,
                    u64& kept_w) -> u64 {
    while (true) {
      if (in_cnt <= kList) return order_list(key_lo, key_hi, by_weight, target, base_cnt, base_w, kept_w);
      if (key_lo == key_hi) {
        // more equal keys than the list holds: the m-th of them in index order is the last kept
        const uint32_t w = weight(__uint_as_float(key_lo));
        const u64 m = by_weight ? (target - base_w + w - 1) / max(w, 1u) : target - base_cnt;
        kept_w = base_w + m * w;
        u64 cnt = 0, warp_cnt, ahead, ties;
        for (int i = s0 + lane; i < s1; i += 32) cnt += xkey[i] == key_lo;
        sum_over(cnt, 1, warp_cnt, ahead, ties);
        if (ahead < m && ahead + warp_cnt >= m) {
          for (int base = s0; base < s1; base += 32) {
            const int i = base + lane;
            const uint32_t hit = __ballot_sync(0xffffffffu, i < s1 && xkey[i] == key_lo);
            const int c = __popc(hit);
            if (ahead + c >= m) {
              const int nth = int(m - ahead);   // 1-based among the hits of these 32
              if ((hit >> lane & 1) && __popc(hit & ((2u << lane) - 1)) == nth) {
                const u64 id = (u64(key_lo) << 32) | uint32_t(lo + i);
                for (int r = 0; r < C; ++r) *cluster.map_shared_rank(&S.found, r) = id;
              }
              break;
            }
            ahead += c;
          }
        }
        publish();
        const u64 id = S.found;
        publish();
        return id;
      }
      publish();               // every CTA has read the previous histogram
      dirty = true;
      clear();
      __syncthreads();
      int shift = 0;
      while (((key_hi - key_lo) >> shift) >= kBins) ++shift;
      for (int i = s0 + lane; i < s1; i += 32) {
        const uint32_t key = xkey[i];
        if (key >= key_lo && key <= key_hi) add_to_bin((key - key_lo) >> shift, weight(x[i]));
      }
      publish();
      find_bin(by_weight, target, base_cnt, base_w);
      if (S.found_bin < 0) return kAll;   // (the range always holds the crossing)
      base_cnt = S.found_cnt;
      base_w = S.found_w;
      in_cnt = S.found_in_cnt;
      key_lo += uint32_t(S.found_bin) << shift;
      key_hi = min(key_hi, key_lo + ((1u << shift) - 1));
    }
  };
  __syncthreads();
  if (by_k && use_p) {         // top-p needs the kept weight: sums beside the counts
    fill_all();
    find_bin(false, limit, 0, 0);
    bin = S.found_bin;
    bin_cnt = S.found_cnt;
    bin_w = S.found_w;
    bin_in = S.found_in_cnt;
    __syncthreads();
  }
  if (cut_somewhere && bin >= 0) {
    u64 total_k;
    cut = refine(first_lo(bin), first_lo(bin + 1) - 1, !by_k, limit, bin_cnt, bin_w, bin_in, total_k);
    if (by_k && use_p) {
      // top-p among the tokens that top-k kept
      limit = max(share(total_k, top_p), u64(1));
      if (dirty) fill_all();
      else publish();
      find_bin(true, limit, 0, 0);
      const int p_bin = S.found_bin;
      const u64 p_cnt = S.found_cnt, p_w = S.found_w, p_in = S.found_in_cnt;
      __syncthreads();
      u64 unused;
      if (p_bin >= 0) cut = min(cut, refine(first_lo(p_bin), first_lo(p_bin + 1) - 1, true, limit, p_cnt, p_w, p_in, unused));
    }
  }
  const uint32_t cut_key = uint32_t(cut >> 32);
  auto kept = [&](int i) -> uint32_t {
    const float d = x[i];
    const uint32_t key = __float_as_uint(d);
    if (key > cut_key) return 0u;
    const uint32_t w = weight(d);
    return (((u64(key) << 32) | uint32_t(lo + i)) <= cut && w >= min_w) ? w : 0u;
  };
  sum = 0;
  for (int i = s0 + lane; i < s1; i += 32) sum += kept(i);
  __syncthreads();
  publish();                   // slot[0] has been read everywhere
  sum_over(sum, 0, mine, below, total);   // its barrier: the last access to another CTA's memory is behind it
  draw(kept, mine, below, total);
}

template <bool BF16>
cudaError_t launch(const SampleArgs& a, int cluster, int slice, cudaStream_t s) {
  auto bytes = [](int c, int n) { return sizeof(Shared) + size_t(kBins / c) * 12 + size_t(n) * sizeof(float); };
  const size_t smem = bytes(cluster, slice);
  auto kernel = sample_kernel<BF16>;
  cudaError_t e = once_per_device_kernel(reinterpret_cast<const void*>(kernel), [&] {
    cudaError_t r = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         int(std::max(bytes(8, kMaxSlice), bytes(1, kPairSlice))));
    if (r == cudaSuccess) r = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    return r;
  });
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(a.B) * unsigned(cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(cluster);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, a, slice);
}

}  // namespace

const char* sample(const SampleArgs& a, cudaStream_t s) {
  if (a.B < 1) return nullptr;
  if (a.V < 1) return "sample: no tokens";
  if (a.V > kMaxCluster * kMaxSlice) return "sample: at most 720896 tokens a row";
  if ((long)a.B * kMaxCluster > 0x7fffffffl) return "sample: too many rows";
  // CTAs a row: enough that two of them fit an SM (16 are the limit: longer slices beyond), and twice as
  // many while all rows' still run at once, two an SM. 151936 tokens with 8 and 16 CTAs a row: 24.6 and
  // 20.5 us for 1 row, 55 and 47 for 18, 55 and 74 for 37, 115 and 174 for 129; with 4: 29, 64, 68, 139.
  int cluster = 1;
  while (cluster < 8 && cluster * kPairSlice < a.V) cluster *= 2;   // (one CTA: 20480 tokens at most)
  while (cluster < kMaxCluster && cluster * kMaxSlice < a.V) cluster *= 2;
  while (cluster < kMaxCluster && (long)cluster * a.B <= a.num_sms && a.V / (2 * cluster) >= 2048) cluster *= 2;
  const int slice = ((a.V + cluster - 1) / cluster + 7) / 8 * 8;
  const cudaError_t e = a.bf16 ? launch<true>(a, cluster, slice, s) : launch<false>(a, cluster, slice, s);
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace sampling
}  // namespace hcp
