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
// are read from memory once. The k-th and the top-p cut are found by a histogram over d (bins of
// 1/64, counts and weight sums, summed over the cluster through distributed shared memory), then
// exactly among the few tokens of the crossing bin. Bound: the chain of block and cluster barriers
// for a few rows, the shared-memory passes and atomics for many.
#include <cooperative_groups.h>

#include <cuda_bf16.h>

#include "common.cuh"
#include "launch.h"
#include "sample.h"

namespace hcp {
namespace sampling {

using namespace hcp::dev;
namespace cg = cooperative_groups;

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kList = 512;          // tokens of a crossing bin that are ordered directly
constexpr int kMaxCluster = 16;     // 16 is the hardware's limit (above 8: opt-in)
constexpr int kMaxSlice = 45056;    // floats of a row in one CTA's shared memory
constexpr u64 kAll = ~0ull;

// The fixed operations of the weight: no contraction, no flush of subnormals, whatever the flags.
__device__ __forceinline__ float mul_rn(float a, float b) {
  float r;
  asm("mul.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float add_rn(float a, float b) {
  float r;
  asm("add.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float div_rn(float a, float b) {
  float r;
  asm("div.rn.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// floor(2^31 exp(-d)) for 0 <= d <= 64: y = d log2(e), n = round(y), 2^(n - y) on [-1/2, 1/2] by the
// Taylor series of 2^g to degree 7 (remainder below 1e-8), then a shift by n.
__device__ __forceinline__ uint32_t weight(float d) {
  const float y = mul_rn(d, 0x1.715476p+0f);
  const float n = rintf(y);
  const float g = add_rn(n, -y);
  float w = 0x1.ffcbfcp-17f;
  w = add_rn(mul_rn(w, g), 0x1.430912p-13f);
  w = add_rn(mul_rn(w, g), 0x1.5d87fep-10f);
  w = add_rn(mul_rn(w, g), 0x1.3b2ab6p-7f);
  w = add_rn(mul_rn(w, g), 0x1.c6b08ep-5f);
  w = add_rn(mul_rn(w, g), 0x1.ebfbep-3f);
  w = add_rn(mul_rn(w, g), 0x1.62e43p-1f);
  w = add_rn(mul_rn(w, g), 1.0f);
  const uint32_t fix = __float2uint_rz(w * 2147483648.f);
  const int sh = int(n);
  return sh > 31 ? 0u : fix >> sh;
}

__device__ __forceinline__ int bin_of(float d) { return min(int(d * 64.f), kBins - 1); }

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

struct Shared {
  uint32_t cnt[kBins], wlo[kBins], whi[kBins];   // this CTA's histogram
  u64 list[kList];                               // this CTA's tokens of the crossing bin
  u64 all[kList];                                // the cluster's
  u64 warp_a[kWarps], warp_b[kWarps];
  u64 slot[2][kMaxCluster];                      // one value of every CTA, pushed by it
  float fslot[kMaxCluster];
  int list_n;
  u64 found;                                     // results one thread hands to the block
  u64 found_cnt, found_w, found_in_cnt, found_in_w;
  int found_bin;
};

template <bool BF16>
__global__ void __launch_bounds__(kThreads, 1) sample_kernel(SampleArgs a, int slice) {
  extern __shared__ __align__(16) unsigned char raw[];
  Shared& S = *reinterpret_cast<Shared*>(raw);
  float* x = reinterpret_cast<float*>(raw + sizeof(Shared));
  cg::cluster_group cluster = cg::this_cluster();
  const int C = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int b = blockIdx.x / C;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
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
    for (int i = tid; i < nv; i += kThreads) {
      const uint4 v = ld_nc_v4(src + (long)i * 16);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (BF16) {
          float f0 = bf16_lo(w[j]), f1 = bf16_hi(w[j]);
          f0 = f0 == f0 ? f0 : ninf;
          f1 = f1 == f1 ? f1 : ninf;
          x[i * 8 + 2 * j] = f0;
          x[i * 8 + 2 * j + 1] = f1;
          top = fmaxf(top, fmaxf(f0, f1));
        } else {
          float f = __uint_as_float(w[j]);
          f = f == f ? f : ninf;
          x[i * 4 + j] = f;
          top = fmaxf(top, f);
        }
      }
    }
    for (int i = nv * vec + tid; i < n; i += kThreads) {
      float f = BF16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(src)[i])
                     : reinterpret_cast<const float*>(src)[i];
      f = f == f ? f : ninf;
      x[i] = f;
      top = fmaxf(top, f);
    }
  }
  const float temp = a.temperature.ptr ? a.temperature.ptr[b] : a.temperature.value;
  const int top_k = a.top_k.ptr ? a.top_k.ptr[b] : a.top_k.value;
  const float top_p = a.top_p.ptr ? a.top_p.ptr[b] : a.top_p.value;
  const float min_p = a.min_p.ptr ? a.min_p.ptr[b] : a.min_p.value;
  const bool greedy = !(temp > 0.f);
  const bool use_k = !greedy && top_k > 0 && top_k < a.V;
  const bool use_p = !greedy && top_p > 0.f && top_p < 1.f;
  if (use_k || use_p) {
    for (int i = tid; i < kBins; i += kThreads) S.cnt[i] = S.wlo[i] = S.whi[i] = 0;
  }
  if (tid == 0) S.list_n = 0;
  top = warp_max(top);
  float* wf = reinterpret_cast<float*>(S.warp_a);
  if (lane == 0) wf[warp] = top;
  cluster.sync();      // every CTA of the cluster runs: its shared memory may be written
  top = warp_max(wf[lane]);
  if (tid < C) *cluster.map_shared_rank(&S.fslot[rank], tid) = top;
  cluster.sync();
  top = S.fslot[0];
  for (int i = 1; i < C; ++i) top = fmaxf(top, S.fslot[i]);

  if (top == ninf) {   // nothing to draw (the whole cluster agrees)
    if (rank == 0 && tid == 0) a.token[b] = -1;
    return;
  }
  if (greedy) {
    uint32_t best = 0xffffffffu;
    for (int i = s0 + lane; i < s1; i += 32)
      if (x[i] == top) best = min(best, uint32_t(lo + i));
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

  // ---------------------------------------------------------------- distances, totals, histogram
  auto add_to_bin = [&](int bin, uint32_t w) {
    atomicAdd(&S.cnt[bin], 1u);
    if (w) {
      const uint32_t was = atomicAdd(&S.wlo[bin], w);
      if (was + w < was) atomicAdd(&S.whi[bin], 1u);   // the carry of a 64-bit sum
    }
  };
  u64 sum = 0;
  for (int i = s0 + lane; i < s1; i += 32) {
    const float l = x[i];
    float d = l == top ? 0.f : div_rn(top - l, temp);
    d = d == d ? fminf(d, 64.f) : 64.f;
    x[i] = d;
    const uint32_t w = weight(d);
    sum += w;
    if (use_k || use_p) add_to_bin(bin_of(d), w);
  }

  u64 cut = kAll;
  if (use_k || use_p) {
    const uint32_t* xkey = reinterpret_cast<const uint32_t*>(x);
    // Finds the (key, index) of the last kept token of a prefix search, the prefix's weight
    // included in `kept_w`. Levels: the histogram in place covers keys [key_lo, key_hi] with
    // `shift` (the first level: d in bins of 1/64); a crossing bin of at most kList tokens is
    // ordered directly, a larger one gets a histogram of its own.
    u64 limit_id = kAll;     // top-p looks at the tokens that top-k kept
    bool dirty = false;      // the first level's histogram has been overwritten
    auto publish = [&] { cluster.sync(); };
    auto find_bin = [&](bool by_weight, u64 target, u64 base_cnt, u64 base_w) {
      // sums of two bins a thread over the cluster, then a block scan to the crossing bin
      u64 c[2] = {0, 0}, w[2] = {0, 0};
      for (int r = 0; r < C; ++r) {
        const Shared* o = cluster.map_shared_rank(&S, r);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int bin = 2 * tid + j;
          c[j] += o->cnt[bin];
          w[j] += (u64(o->whi[bin]) << 32) + o->wlo[bin];
        }
      }
      u64 ic = c[0] + c[1], iw = w[0] + w[1];
      const u64 oc = ic, ow = iw;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const u64 uc = __shfl_up_sync(0xffffffffu, ic, d), uw = __shfl_up_sync(0xffffffffu, iw, d);
        if (lane >= d) {
          ic += uc;
          iw += uw;
        }
      }
      if (tid == 0) S.found_bin = -1;
      if (lane == 31) {
        S.warp_a[warp] = ic;
        S.warp_b[warp] = iw;
      }
      __syncthreads();
      u64 ec = base_cnt + ic - oc, ew = base_w + iw - ow;
      for (int i = 0; i < warp; ++i) {
        ec += S.warp_a[i];
        ew += S.warp_b[i];
      }
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const u64 before = by_weight ? ew : ec, in = by_weight ? w[j] : c[j];
        if (before < target && before + in >= target) {
          S.found_bin = 2 * tid + j;
          S.found_cnt = ec;
          S.found_w = ew;
          S.found_in_cnt = c[j];
          S.found_in_w = w[j];
        }
        ec += c[j];
        ew += w[j];
      }
      __syncthreads();
    };
    // Among the tokens whose key lies in [key_lo, key_hi] (all of them in the list): the last
    // kept one. `before`: count or weight ahead of the list.
    auto order_list = [&](uint32_t key_lo, uint32_t key_hi, bool by_weight, u64 target, u64 base_cnt, u64 base_w,
                          u64& kept_w) {
      for (int i = s0 + lane; i < s1; i += 32) {
        const uint32_t key = xkey[i];
        if (key >= key_lo && key <= key_hi) {
          const int at = atomicAdd(&S.list_n, 1);
          if (at < kList) S.list[at] = (u64(key) << 32) | uint32_t(lo + i);
        }
      }
      publish();
      int total = 0;
      for (int r = 0; r < C; ++r) {
        const Shared* o = cluster.map_shared_rank(&S, r);
        const int m = min(o->list_n, kList);
        for (int i = tid; i < m && total + i < kList; i += kThreads) S.all[total + i] = o->list[i];
        total = min(total + m, kList);
      }
      if (tid == 0) {
        S.found = kAll;
        S.found_w = 0;
      }
      __syncthreads();
      // one thread a token: what is ahead of it decides
      if (tid < total) {
        const u64 me = S.all[tid];
        u64 cnt = base_cnt, w = base_w;
        for (int i = 0; i < total; ++i) {
          const u64 o = S.all[i];
          if (o < me) {
            ++cnt;
            w += weight(__uint_as_float(uint32_t(o >> 32)));
          }
        }
        const u64 own = weight(__uint_as_float(uint32_t(me >> 32)));
        const u64 before = by_weight ? w : cnt, in = by_weight ? own : 1;
        if (before < target && before + in >= target) {
          S.found = me;
          S.found_w = w + own;
        }
      }
      publish();             // also: every CTA has read the lists
      if (tid == 0) S.list_n = 0;
      kept_w = S.found_w;
      const u64 id = S.found;
      __syncthreads();
      return id;
    };
    // The crossing bin at `shift` levels below the first; fills a new histogram of [key_lo, key_hi].
    auto refine = [&](uint32_t key_lo, uint32_t key_hi, bool by_weight, u64 target, u64 base_cnt, u64 base_w,
                      u64 in_cnt, u64& kept_w) -> u64 {
      while (true) {
        if (in_cnt <= kList) return order_list(key_lo, key_hi, by_weight, target, base_cnt, base_w, kept_w);
        if (key_lo == key_hi) {
          // more equal keys than the list holds: the m-th of them in index order is the last kept
          const uint32_t w = weight(__uint_as_float(key_lo));
          u64 m = by_weight ? (target - base_w + w - 1) / max(w, 1u) : target - base_cnt;
          kept_w = base_w + m * w;
          u64 cnt = 0;
          for (int i = s0 + lane; i < s1; i += 32) cnt += xkey[i] == key_lo;
          cnt = warp_sum64(cnt);
          if (lane == 0) S.warp_a[warp] = cnt;
          __syncthreads();
          if (tid == 0) {
            u64 t = 0;
            for (int i = 0; i < kWarps; ++i) t += S.warp_a[i];
            for (int r = 0; r < C; ++r) *cluster.map_shared_rank(&S.slot[1][rank], r) = t;
          }
          publish();
          u64 ahead = 0, mine = 0;
          int owner = C - 1;
          for (int r = 0; r < C; ++r) {
            if (ahead + S.slot[1][r] >= m) {
              owner = r;
              break;
            }
            ahead += S.slot[1][r];
          }
          mine = ahead;
          if (owner == rank) {
            for (int i = 0; i < warp; ++i) mine += S.warp_a[i];
            if (mine < m && mine + S.warp_a[warp] >= m) {
              for (int base = s0; base < s1; base += 32) {
                const int i = base + lane;
                const uint32_t hit = __ballot_sync(0xffffffffu, i < s1 && xkey[i] == key_lo);
                const int c = __popc(hit);
                if (mine + c >= m) {
                  const int nth = int(m - mine);   // 1-based among the hits of these 32
                  if ((hit >> lane & 1) && __popc(hit & ((2u << lane) - 1)) == nth) {
                    const u64 id = (u64(key_lo) << 32) | uint32_t(lo + i);
                    for (int r = 0; r < C; ++r) *cluster.map_shared_rank(&S.found, r) = id;
                  }
                  break;
                }
                mine += c;
              }
            }
          }
          publish();
          const u64 id = S.found;
          publish();
          return id;
        }
        publish();           // every CTA has read the previous histogram
        dirty = true;
        for (int i = tid; i < kBins; i += kThreads) S.cnt[i] = S.wlo[i] = S.whi[i] = 0;
        __syncthreads();
        int shift = 0;
        while (((key_hi - key_lo) >> shift) >= kBins) ++shift;
        for (int i = s0 + lane; i < s1; i += 32) {
          const uint32_t key = xkey[i];
          if (key >= key_lo && key <= key_hi) {
            add_to_bin((key - key_lo) >> shift, weight(x[i]));
          }
        }
        publish();
        find_bin(by_weight, target, base_cnt, base_w);
        if (S.found_bin < 0) return kAll;   // (the range always holds the crossing)
        base_cnt = S.found_cnt;
        base_w = S.found_w;
        in_cnt = S.found_in_cnt;
        key_lo += uint32_t(S.found_bin) << shift;
        key_hi = min(key_hi, key_lo + ((1u << shift) - 1));
        __syncthreads();
      }
    };
    // The first level's bin b holds the keys with floor(64 d) == b.
    auto first_lo = [](int bin) { return __float_as_uint(float(bin) * (1.f / 64.f)); };

    publish();               // the histograms are complete
    u64 total_k = 0;
    bool whole = true;       // top-k keeps every token with a weight
    if (use_k) {
      find_bin(false, u64(top_k), 0, 0);
      const int bin = S.found_bin;
      const u64 bc = S.found_cnt, bw = S.found_w, ic = S.found_in_cnt;
      __syncthreads();
      // the last bin holds only weights of 0: a cut inside it leaves the draw as it is
      if (bin >= 0 && bin < kBins - 1) {
        whole = false;
        cut = refine(first_lo(bin), first_lo(bin + 1) - 1, false, u64(top_k), bc, bw, ic, total_k);
        limit_id = cut;
      }
    }
    if (use_p) {
      if (whole) {
        u64 t = warp_sum64(sum);
        if (lane == 0) S.warp_a[warp] = t;
        __syncthreads();
        t = warp_sum64(S.warp_a[lane]);
        if (tid < C) *cluster.map_shared_rank(&S.slot[0][rank], tid) = t;
        publish();
        for (int r = 0; r < C; ++r) total_k += S.slot[0][r];
      }
      const u64 target = max(share(total_k, top_p), u64(1));
      if (dirty) {
        publish();
        for (int i = tid; i < kBins; i += kThreads) S.cnt[i] = S.wlo[i] = S.whi[i] = 0;
        __syncthreads();
        for (int i = s0 + lane; i < s1; i += 32) add_to_bin(bin_of(x[i]), weight(x[i]));
        publish();
      }
      find_bin(true, target, 0, 0);
      const int bin = S.found_bin;
      const u64 bc = S.found_cnt, bw = S.found_w, ic = S.found_in_cnt;
      __syncthreads();
      if (bin >= 0) {
        u64 unused;
        cut = min(limit_id, refine(first_lo(bin), first_lo(bin + 1) - 1, true, target, bc, bw, ic, unused));
      }
    }
    publish();               // shared slots may be reused
  }

  // ---------------------------------------------------------------- the draw
  const uint32_t min_w = min_p > 0.f ? uint32_t(fminf(min_p, 1.f) * 2147483648.f) : 0u;
  auto kept = [&](int i) -> uint32_t {
    const float d = x[i];
    const uint32_t w = weight(d);
    const u64 id = (u64(__float_as_uint(d)) << 32) | uint32_t(lo + i);
    return (id <= cut && w >= min_w) ? w : 0u;
  };
  sum = 0;
  for (int i = s0 + lane; i < s1; i += 32) sum += kept(i);
  sum = warp_sum64(sum);
  __syncthreads();
  if (lane == 0) S.warp_a[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    const u64 t = warp_sum64(S.warp_a[lane]);
    if (lane < C) *cluster.map_shared_rank(&S.slot[0][rank], lane) = t;
  }
  cluster.sync();            // the last access to another CTA's shared memory is behind it
  u64 total = 0, ahead = 0;
  for (int r = 0; r < C; ++r) {
    if (r < rank) ahead += S.slot[0][r];
    total += S.slot[0][r];
  }
  const float u = a.u[b];
  const u64 target = share(total, fminf(u, 0.99999994f));
  for (int i = 0; i < warp; ++i) ahead += S.warp_a[i];
  if (target >= ahead && target < ahead + sum) {
    for (int base = s0; base < s1; base += 32) {
      const int i = base + lane;
      u64 inc = i < s1 ? kept(i) : 0u;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const u64 up = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += up;
      }
      const uint32_t hit = __ballot_sync(0xffffffffu, ahead + inc > target);
      if (hit) {
        if (lane == __ffs(hit) - 1) a.token[b] = lo + i;
        break;
      }
      ahead += __shfl_sync(0xffffffffu, inc, 31);
    }
  }
}

template <bool BF16>
cudaError_t launch(const SampleArgs& a, int cluster, int slice, cudaStream_t s) {
  const size_t smem = sizeof(Shared) + size_t(slice) * sizeof(float);
  auto kernel = sample_kernel<BF16>;
  cudaError_t e = once_per_device_kernel(reinterpret_cast<const void*>(kernel), [&] {
    cudaError_t r = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         int(sizeof(Shared) + kMaxSlice * sizeof(float)));
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
  // CTAs a row: enough to hold it, and more while there are SMs without a row
  int cluster = 1;
  while (cluster * kMaxSlice < a.V) cluster *= 2;
  while (cluster < 8 && 2l * cluster * a.B <= a.num_sms && a.V / (2 * cluster) >= 2048) cluster *= 2;
  const int slice = ((a.V + cluster - 1) / cluster + 7) / 8 * 8;
  const cudaError_t e = a.bf16 ? launch<true>(a, cluster, slice, s) : launch<false>(a, cluster, slice, s);
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace sampling
}  // namespace hcp
