// Block tables and slot maps of one step, built on the GPU from request lengths.
//
// Row r grows by n_r = add[r] tokens (or, negative, gives its pages back). With P tokens a page:
//   need_r = ceil((old_r + n_r) / P) - ceil(old_r / P)    pages taken from the FIFO ring, in row order
//   slot(t) = table[r][p / P] * P + p % P                 for the token at position p of row r
// and a "unit" per block that the new tokens touch, the work list of the append. A step that does
// not fit (tokens, table width, free pages, or more pages given back than the ring has places for)
// changes nothing and says so in info[3].
//
// Bound: latency. The arrays are a few bytes per row and token, so one launch does the whole step:
// every CTA scans all rows (four sums at once) and the CTAs share the tokens, units and pages to
// write. New pages are looked up by their place in the ring rather than through the table, so no CTA
// depends on an entry that another one writes. Where the new lengths or counters overwrite the old
// ones, the CTAs form one cluster (of at most 8) whose barrier separates the reads of the state from
// its update; otherwise there are as many CTAs as the writes are worth. Measured on B200, caches cold:
// 64 rows growing by a token 10 us with 1 to 64 CTAs; 509 rows with 131072 new tokens (2 MB written)
// 135 us with one CTA, 25 with 8, 14 with 32 or more.
#include <cooperative_groups.h>

#include "common.cuh"
#include "launch.h"
#include "paged8.h"

namespace hcp {
namespace kv8 {

using namespace hcp::dev;
namespace cg = cooperative_groups;

namespace {

struct Sums {
  long long n;  // tokens (64 bits: lengths are the caller's)
  int units, need, back;
  __device__ __forceinline__ Sums operator+(const Sums& o) const {
    return {n + o.n, units + o.units, need + o.need, back + o.back};
  }
};

__device__ __forceinline__ Sums shfl_up(const Sums& v, int d) {
  return {__shfl_up_sync(0xffffffffu, v.n, d), __shfl_up_sync(0xffffffffu, v.units, d),
          __shfl_up_sync(0xffffffffu, v.need, d), __shfl_up_sync(0xffffffffu, v.back, d)};
}

// Largest r in [0, n) with off[r] <= x, off ascending and off[0] <= x.
__device__ __forceinline__ int find_row(const int* off, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (off[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// x mod n for x >= 0, in 32 bits where they hold it.
__device__ __forceinline__ int modulo(long long x, int n) {
  x = x < 0 ? 0 : x;
  return (x >> 32) == 0 ? int(uint32_t(x) % uint32_t(n)) : int(x % n);
}

// SHIFT: the page size is 1 << a.shift. CLUSTER: the new state may overwrite the old one.
template <bool SHIFT, bool CLUSTER>
__global__ void __launch_bounds__(1024) plan_kernel(PlanArgs a) {
  extern __shared__ int sm[];
  int* s_cu = sm;                      // [R + 1] first token of each row
  int* s_unit = s_cu + a.R + 1;        // [R + 1] first unit
  int* s_need = s_unit + a.R + 1;      // [R + 1] first page taken
  int* s_back = s_need + a.R + 1;      // [R + 1] first page given back
  int* s_old = s_back + a.R + 1;       // [R]
  __shared__ Sums warp_tot[32];
  const int tid = threadIdx.x, nth = blockDim.x, lane = tid & 31, warp = tid >> 5;
  pdl_trigger();
  pdl_wait();

  const int P = a.P;
  auto pages_before = [&](int x) { return SHIFT ? x >> a.shift : x / P; };      // whole pages below position x
  auto pages_for = [&](int x) { return SHIFT ? (x + P - 1) >> a.shift : (x + P - 1) / P; };
  const long long cap = (long long)a.width * P;
  const int per = (a.R + nth - 1) / nth;
  const int r0 = min(a.R, tid * per), r1 = min(a.R, r0 + per);
  const long long head = a.counters[0], tail = a.counters[1];
  Sums own{0, 0, 0, 0};
  bool wide = false;
  auto row_of = [&](int r, int& old) {
    const int add = a.add[r];
    old = int(min((long long)max(a.kv_len[r], 0), cap));
    const int have = pages_for(old);
    Sums v{0, 0, 0, 0};
    if (add < 0) {
      v.back = have;
    } else if (add > 0) {
      const long long end = (long long)old + add;
      if (end > cap) {
        wide = true;
      } else {
        v.need = pages_for(int(end)) - have;
        v.units = pages_for(int(end)) - pages_before(old);
      }
      v.n = add;
    }
    return v;
  };
  for (int r = r0; r < r1; ++r) {
    int old;
    own = own + row_of(r, old);
  }
  // inclusive scan over the block
  Sums inc = own;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const Sums up = shfl_up(inc, d);
    if (lane >= d) inc = inc + up;
  }
  if (lane == 31) warp_tot[warp] = inc;
  const bool any_wide = __syncthreads_or(wide);
  Sums total = lane < nth / 32 ? warp_tot[lane] : Sums{0, 0, 0, 0};
  const Sums own_warp = total;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const Sums up = shfl_up(total, d);
    if (lane >= d) total = total + up;
  }
  Sums before{__shfl_sync(0xffffffffu, total.n - own_warp.n, warp), __shfl_sync(0xffffffffu, total.units - own_warp.units, warp),
              __shfl_sync(0xffffffffu, total.need - own_warp.need, warp), __shfl_sync(0xffffffffu, total.back - own_warp.back, warp)};
  total = Sums{__shfl_sync(0xffffffffu, total.n, 31), __shfl_sync(0xffffffffu, total.units, 31),
               __shfl_sync(0xffffffffu, total.need, 31), __shfl_sync(0xffffffffu, total.back, 31)};
  Sums ex{before.n + inc.n - own.n, before.units + inc.units - own.units, before.need + inc.need - own.need,
          before.back + inc.back - own.back};
  const long long avail = min(max(tail - head, 0ll), (long long)a.ring_size);
  int status = 0;
  if (total.n > a.max_tokens) status = 3;
  else if (any_wide) status = 2;
  else if (total.need > avail + total.back) status = 1;
  else if (avail + total.back > a.ring_size) status = 4;   // (the writes to the ring below rely on it)
  const bool ok = status == 0;
  if (!ok) total = Sums{0, 0, 0, 0};
  for (int r = r0; r < r1; ++r) {
    int old;
    const Sums v = row_of(r, old);
    s_cu[r] = ok ? int(ex.n) : 0;
    s_unit[r] = ok ? ex.units : 0;
    s_need[r] = ok ? ex.need : 0;
    s_back[r] = ok ? ex.back : 0;
    s_old[r] = old;
    ex = ex + v;
  }
  if (tid == 0) {
    s_cu[a.R] = int(total.n);
    s_unit[a.R] = total.units;
    s_need[a.R] = total.need;
    s_back[a.R] = total.back;
  }
  // the state has been read by every CTA that will: it may be overwritten from here on
  if (CLUSTER) cg::this_cluster().sync();
  else __syncthreads();

  const int T = int(total.n), U = total.units;
  const int crank = blockIdx.x, csize = gridDim.x;
  const int gtid = crank * nth + tid, gn = csize * nth;
  const long long size = a.ring_size;
  const int head_at = modulo(head, a.ring_size), tail_at = modulo(tail, a.ring_size);
  // page i of those taken in this step: first the ring's, then the ones given back in this step
  auto taken = [&](int i) {
    if (i < avail) {
      long long at = (long long)head_at + i;
      return a.ring[at >= size ? at - size : at];
    }
    const int j = i - int(avail);
    const int r = find_row(s_back, a.R, j);
    return a.table[(long)r * a.width + (j - s_back[r])];
  };
  auto page_of = [&](int r, int block) {
    const int have = pages_for(s_old[r]);
    return block < have ? a.table[(long)r * a.width + block] : taken(s_need[r] + block - have);
  };

  if (crank == 0) {
    for (int r = tid; r < a.R; r += nth) {
      const int n = s_cu[r + 1] - s_cu[r];
      a.cu[r] = s_cu[r];
      a.kv_len_out[r] = (ok && s_back[r + 1] != s_back[r]) ? 0 : s_old[r] + n;
    }
    if (tid == 0) {
      a.cu[a.R] = T;
      a.info[0] = T;
      a.info[1] = U;
      a.info[2] = total.need;
      a.info[3] = status;
      a.counters_out[0] = head + total.need;
      a.counters_out[1] = tail + total.back;
    }
  }
  // slot map: four tokens a thread, so that every array is written in 16-byte pieces
  const int quads = (a.max_tokens + 3) / 4;
  for (int i = gtid; i < quads; i += gn) {
    int row[4], pos[4];
    long long slot[4];
    const int t0 = 4 * i;
    int r = t0 < T ? find_row(s_cu, a.R + 1, t0) : 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = t0 + j;
      row[j] = -1;
      pos[j] = 0;
      slot[j] = -1;
      if (t < T) {
        while (s_cu[r + 1] <= t) ++r;
        const int p = s_old[r] + t - s_cu[r];
        row[j] = r;
        pos[j] = p;
        const int block = pages_before(p);
        slot[j] = (long long)page_of(r, block) * P + (p - block * P);
      }
    }
    if (t0 + 4 <= a.max_tokens) {
      reinterpret_cast<int4*>(a.row)[i] = make_int4(row[0], row[1], row[2], row[3]);
      reinterpret_cast<int4*>(a.pos)[i] = make_int4(pos[0], pos[1], pos[2], pos[3]);
      reinterpret_cast<longlong2*>(a.slot)[2 * i] = make_longlong2(slot[0], slot[1]);
      reinterpret_cast<longlong2*>(a.slot)[2 * i + 1] = make_longlong2(slot[2], slot[3]);
    } else {
      for (int j = 0; t0 + j < a.max_tokens; ++j) {
        a.row[t0 + j] = row[j];
        a.pos[t0 + j] = pos[j];
        a.slot[t0 + j] = slot[j];
      }
    }
  }
  for (int i = gtid; i < a.max_units; i += gn) {
    int4 u = make_int4(-1, 0, 0, 0);
    if (i < U) {
      const int r = find_row(s_unit, a.R + 1, i);
      const int old = s_old[r], end = old + s_cu[r + 1] - s_cu[r];
      const int block = pages_before(old) + i - s_unit[r];
      const int p0 = max(block * P, old), p1 = min((block + 1) * P, end);
      u = make_int4(r, s_cu[r] + p0 - old, p1 - p0, p0);
    }
    a.unit[i] = u;
  }
  for (int i = gtid; i < total.need; i += gn) {
    const int r = find_row(s_need, a.R + 1, i);
    a.table[(long)r * a.width + pages_for(s_old[r]) + i - s_need[r]] = taken(i);
  }
  for (int i = gtid; i < total.back; i += gn) {
    const int r = find_row(s_back, a.R + 1, i);
    const long long at = (long long)tail_at + i;
    a.ring[at >= size ? at - size : at] = a.table[(long)r * a.width + i - s_back[r]];
  }
}

}  // namespace

namespace {

template <bool SHIFT, bool CLUSTER>
cudaError_t launch(const PlanArgs& a, int ctas, int threads, cudaStream_t s) {
  auto kernel = plan_kernel<SHIFT, CLUSTER>;
  cudaError_t e = once_per_device_kernel(reinterpret_cast<const void*>(kernel), [&] {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (5 * kPlanMaxRows + 8) * int(sizeof(int)));
  });
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(ctas));
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = (size_t(a.R + 1) * 4 + a.R) * sizeof(int);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (CLUSTER) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = unsigned(ctas);
    attr[n].val.clusterDim.y = 1;
    attr[n++].val.clusterDim.z = 1;
  }
  cfg.attrs = attr;
  cfg.numAttrs = unsigned(n);
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

}  // namespace

const char* plan_step(const PlanArgs& args, cudaStream_t s) {
  PlanArgs a = args;
  if (a.R < 1 || a.R > kPlanMaxRows) return "plan_step: 1 to 4096 rows";
  if (a.P < 1 || a.width < 1 || a.ring_size < 1) return "plan_step: empty table, ring or page";
  if ((long long)a.R * a.width >= (1ll << 31) || (long long)a.width * a.P >= (1ll << 30))
    return "plan_step: table too large";
  if (a.max_tokens < 1 || a.max_units < 1) return "plan_step: max_tokens and max_units must be positive";
  if (a.max_tokens >= (1 << 30)) return "plan_step: fewer than 2^30 tokens";   // (32-bit token numbers, rounded up to fours)
  // threads for the rows and the token quads of a small step; CTAs for the writes of a large one
  const int quads = (a.max_tokens + 3) / 4;
  const int work = quads > a.max_units ? quads : a.max_units;
  const int most = work > a.R ? work : a.R;
  const int threads = most <= 128 ? 128 : most <= 256 ? 256 : 512;
  const bool in_place = a.kv_len_out == a.kv_len || a.counters_out == a.counters;
  int ctas = 1;
  while (ctas < (in_place ? 8 : 128) && ctas * threads < work) ctas *= 2;
  const bool cluster = in_place && ctas > 1;
  a.shift = 0;
  while ((1 << a.shift) < a.P) ++a.shift;
  const bool shift = (1 << a.shift) == a.P;
  const cudaError_t e = shift ? (cluster ? launch<true, true>(a, ctas, threads, s) : launch<true, false>(a, ctas, threads, s))
                              : (cluster ? launch<false, true>(a, ctas, threads, s) : launch<false, false>(a, ctas, threads, s));
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace kv8
}  // namespace hcp
