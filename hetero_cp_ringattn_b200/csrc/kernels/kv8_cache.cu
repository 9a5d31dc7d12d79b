// Writing and reading back the paged 8-bit KV cache.
//
// rope_append: q and k of every new token are rotated (rotate-half at the token's position), q is
// written out, and k and v are coded into the row's pages. A unit is the run of new tokens inside
// one block of one row; per unit, KV head and k / v the block's scale follows from
//   new block:   s = pow2(amax(new))              open block: s = max(s_old, pow2(amax(new)))
// and when an open block's scale grows, its stored codes are rescaled by s_old / s, a power of
// two. The rotation rounds each product and the sum (no fused multiply-add), and the codes are
// taken from the float32 result, so the codes are reproducible from elementary operations.
//
// gather: the first n cached rows of a request as position-ordered bf16 [Hkv][n][D], the layout
// the prefill attention reads.
//
// Both are bound by memory traffic, the append of a few tokens by latency. Measured on B200 with 32
// query heads, 8 KV heads, 128 dims, pages of 64: append of 16381 tokens 80 us (369 MB, 4.6 TB/s: q's
// half 47 us at 5.7 TB/s, k and v 33 us, their chain of loads, block maximum and codes), of one token
// to each of 64 rows 8 us; gather of 131072 rows 133 us (805 MB, 6.0 TB/s, 92% of a plain copy's rate),
// of 2041 rows with 2 KV heads 6 us.
#include "kv8_common.cuh"
#include "launch.h"

namespace hcp {
namespace kv8 {

using namespace hcp::dev;

namespace {

constexpr int kThreads = 256;

// x1' = x1 c - x2 s, x2' = x2 c + x1 s, every operation rounded by itself.
__device__ __forceinline__ void rotate8(float (&x1)[8], float (&x2)[8], const float (&c)[8], const float (&s)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float a = __fsub_rn(__fmul_rn(x1[j], c[j]), __fmul_rn(x2[j], s[j]));
    const float b = __fadd_rn(__fmul_rn(x2[j], c[j]), __fmul_rn(x1[j], s[j]));
    x1[j] = a;
    x2[j] = b;
  }
}

__device__ __forceinline__ void load_cos_sin(const AppendArgs& a, int pos, int j, float (&c)[8], float (&s)[8]) {
  const long at = (long)pos * (a.c.D / 2) + j;
  load8<kF32>(a.cos_t, at, c);
  load8<kF32>(a.sin_t, at, s);
}

// q of one (token, 8-element chunk) for the heads of a group, whose loads are all in flight before the
// first is used.
constexpr int kQHeads = 4;

template <int DT, int D>
__device__ __forceinline__ void rope_q(const AppendArgs& a, uint32_t item) {
  constexpr int kChunks = D / 16, kAtOnce = DT == kF32 ? (kQHeads + 1) / 2 : kQHeads;
  const int chunk = int(item % kChunks);
  const uint32_t rest = item / kChunks, groups = uint32_t(a.H + kQHeads - 1) / kQHeads;
  const int t = int(rest / groups), h0 = int(rest % groups) * kQHeads;
  if (t >= a.T) return;
  const int pos = a.pos[t];
  const bool ok = pos >= 0 && pos < a.max_pos;
  if (!ok) {   // q of a token without a place is 0
    if (chunk == 0 && h0 == 0) report_error(a.status, int(StatusCode::kOutOfBounds), 401, pos, t);
    for (int h = h0; h < min(a.H, h0 + kQHeads); ++h) {
      uint4* o = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.q_out) + ((long)t * a.H + h) * D + chunk * 8);
      o[0] = o[D / 16] = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  float c[8], s[8];
#pragma unroll
  for (int g = 0; g < kQHeads; g += kAtOnce) {
    Raw8<DT> r1[kAtOnce], r2[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const long at = (long)t * a.row_stride + (long)min(h0 + g + i, a.H - 1) * D + chunk * 8;
      r1[i] = load_raw8<DT>(a.x, at);
      r2[i] = load_raw8<DT>(a.x, at + D / 2);
    }
    if (g == 0) load_cos_sin(a, pos, chunk * 8, c, s);
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int h = h0 + g + i;
      if (h >= a.H) break;
      float x1[8], x2[8];
      floats8<DT>(r1[i], x1);
      floats8<DT>(r2[i], x2);
      rotate8(x1, x2, c, s);
      uint4* o = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.q_out) + ((long)t * a.H + h) * D + chunk * 8);
      o[0] = make_uint4(pack16(a.q_dtype, x1[0], x1[1]), pack16(a.q_dtype, x1[2], x1[3]),
                        pack16(a.q_dtype, x1[4], x1[5]), pack16(a.q_dtype, x1[6], x1[7]));
      o[D / 16] = make_uint4(pack16(a.q_dtype, x2[0], x2[1]), pack16(a.q_dtype, x2[2], x2[3]),
                             pack16(a.q_dtype, x2[4], x2[5]), pack16(a.q_dtype, x2[6], x2[7]));
    }
  }
}

// A unit's place: checked before anything is addressed by it, its positions against the rotary table too.
struct UnitAt {
  int t0, n, p0, start;   // first token, tokens, first position, first offset in the block
  int page;               // -1: nothing to do
};

__device__ __forceinline__ UnitAt unit_at(const AppendArgs& a, uint32_t ui, bool report) {
  UnitAt z{0, 0, 0, 0, -1};
  if (ui >= uint32_t(a.U)) return z;
  const int4 u = a.unit[ui];
  if (u.x < 0) return z;
  const int P = a.c.P, block = u.w / P;
  z.t0 = u.y;
  z.n = u.z;
  z.p0 = u.w;
  z.start = u.w - block * P;
  const bool ok = u.x < a.R && u.y >= 0 && u.z >= 1 && u.z <= a.T - u.y && u.w >= 0 && z.start + u.z <= P && block < a.width &&
                  u.z <= a.max_pos - u.w;
  const int page = ok ? a.table[(long)u.x * a.width + block] : -1;
  if (page >= 0 && page < a.c.pages) z.page = page;
  else if (report) report_error(a.status, int(StatusCode::kOutOfBounds), 402, page, int(ui));
  return z;
}

// 16 values of one (token, chunk): k rotated, v as it is.
template <int DT, int D>
__device__ __forceinline__ void unit_values(const AppendArgs& a, int t, int pos, int col, bool rotate, int chunk, float (&x1)[8],
                                            float (&x2)[8]) {
  const long at = (long)t * a.row_stride + (long)col * D + chunk * 8;
  load8<DT>(a.x, at, x1);
  load8<DT>(a.x, at + D / 2, x2);
  if (rotate) {
    float c[8], s[8];
    load_cos_sin(a, pos, chunk * 8, c, s);
    rotate8(x1, x2, c, s);
  }
}

__device__ __forceinline__ float max_abs(const float (&x1)[8], const float (&x2)[8], float m) {
#pragma unroll
  for (int j = 0; j < 8; ++j) m = fmaxf(m, fmaxf(fabsf(x1[j]), fabsf(x2[j])));
  return m;
}

// 16 stored codes times f (a block whose scale has grown).
template <bool INT8>
__device__ __forceinline__ void rescale16(uint8_t* at, float f) {
  uint4* p = reinterpret_cast<uint4*>(at);
  const uint4 v = *p;
  const uint32_t in[4] = {v.x, v.y, v.z, v.w};
  uint32_t out[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t lo, hi;
    decode4<INT8>(in[j], lo, hi);
    const float2 x = half2_floats(lo), y = half2_floats(hi);
    out[j] = encode4<INT8>(x.x * f, x.y * f, y.x * f, y.y * f);
  }
  *p = make_uint4(out[0], out[1], out[2], out[3]);
}

template <int D, bool INT8>
__device__ __forceinline__ void store_codes(uint8_t* row, int chunk, const float (&x1)[8], const float (&x2)[8], float inv) {
  uint2* p = reinterpret_cast<uint2*>(row + chunk * 8);
  p[0] = make_uint2(encode4<INT8>(x1[0] * inv, x1[1] * inv, x1[2] * inv, x1[3] * inv),
                    encode4<INT8>(x1[4] * inv, x1[5] * inv, x1[6] * inv, x1[7] * inv));
  p[D / 16] = make_uint2(encode4<INT8>(x2[0] * inv, x2[1] * inv, x2[2] * inv, x2[3] * inv),
                         encode4<INT8>(x2[4] * inv, x2[5] * inv, x2[6] * inv, x2[7] * inv));
}

__device__ __forceinline__ float* scale_at(const AppendArgs& a, int kv, int page, int h) {
  return (kv ? a.c.v_scale : a.c.k_scale) + (long)page * a.c.scale_page_stride + (long)h * a.c.scale_head_stride;
}

__device__ __forceinline__ uint8_t* block_at(const AppendArgs& a, int kv, int page, int h) {
  return (kv ? a.c.v : a.c.k) + (long)page * a.c.page_stride + (long)h * a.c.head_stride;
}

// Short units (a decode step): one warp per (unit, KV head, k or v). The first tokens' values stay in
// registers between the maximum and the codes, later ones are read twice.
template <int DT, int D, bool INT8>
__device__ __forceinline__ void store_short(const AppendArgs& a, uint32_t w) {
  constexpr int kChunks = D / 16, kTok = 32 / kChunks;  // tokens a warp covers at a time
  const int lane = threadIdx.x & 31;
  const int kv = int(w & 1);
  const uint32_t rest = w >> 1;
  const int h = int(rest % uint32_t(a.c.Hkv));
  const UnitAt z = unit_at(a, rest / uint32_t(a.c.Hkv), lane == 0);
  if (z.page < 0) return;
  const int chunk = lane % kChunks, sub = lane / kChunks;
  const int col = a.H + (kv ? a.c.Hkv : 0) + h;
  float* sc = scale_at(a, kv, z.page, h);
  const float old = z.start > 0 ? *sc : 0.f;
  float f1[8], f2[8], x1[8], x2[8];
  float amax = 0.f;
  if (sub < z.n) {
    unit_values<DT, D>(a, z.t0 + sub, z.p0 + sub, col, !kv, chunk, f1, f2);
    amax = max_abs(f1, f2, amax);
  }
  for (int i = sub + kTok; i < z.n; i += kTok) {
    unit_values<DT, D>(a, z.t0 + i, z.p0 + i, col, !kv, chunk, x1, x2);
    amax = max_abs(x1, x2, amax);
  }
  amax = warp_max(amax);
  const float scale = fmaxf(old, block_scale<INT8>(amax));
  uint8_t* data = block_at(a, kv, z.page, h);
  if (z.start > 0 && scale > old)
    for (int i = sub; i < z.start; i += kTok) rescale16<INT8>(data + (long)i * a.c.token_stride + chunk * 16, __fdiv_rn(old, scale));
  if (lane == 0) *sc = scale;
  const float inv = __fdiv_rn(1.f, scale);  // exact: a power of two (an old scale may be another value)
  data += (long)z.start * a.c.token_stride;
  if (sub < z.n) store_codes<D, INT8>(data + (long)sub * a.c.token_stride, chunk, f1, f2, inv);
  for (int i = sub + kTok; i < z.n; i += kTok) {
    unit_values<DT, D>(a, z.t0 + i, z.p0 + i, col, !kv, chunk, x1, x2);
    store_codes<D, INT8>(data + (long)i * a.c.token_stride, chunk, x1, x2, inv);
  }
}

// Whole blocks (prompts): P D / 32 threads per (unit, group of KV heads, k or v), 32 values of a head a
// thread held in registers between the maximum and the codes: one pass over the input. The next
// head's loads are in flight while a head is coded, and k's cosines and sines are loaded once.
constexpr int kItems = 2;

__host__ __device__ constexpr int block_threads(int P, int D) { return P * D / 32; }

template <int DT, int D, bool INT8>
__device__ __forceinline__ void store_block(const AppendArgs& a, uint32_t cta, int heads) {
  constexpr int kChunks = D / 16;
  __shared__ float top[2][16];
  const int team = block_threads(a.c.P, D);     // 32 to 512
  const uint32_t w = cta * uint32_t(int(blockDim.x) / team) + uint32_t(int(threadIdx.x) / team);
  const int me = threadIdx.x % team;
  const int kv = int(w & 1);
  const uint32_t rest = w >> 1, groups = uint32_t((a.c.Hkv + heads - 1) / heads);
  const int h0 = int(rest % groups) * heads, h1 = min(a.c.Hkv, h0 + heads);
  const UnitAt z = unit_at(a, rest / groups, me == 0);
  const int n = z.page >= 0 ? z.n : 0;
  const int col0 = a.H + (kv ? a.c.Hkv : 0);
  Raw8<DT> r1[kItems], r2[kItems];
  float c[kItems][8], s[kItems][8];
  auto fetch = [&](int h) {
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int item = k * team + me, i = item / kChunks, chunk = item % kChunks;
      if (i < n) {
        const long at = (long)(z.t0 + i) * a.row_stride + (long)(col0 + h) * D + chunk * 8;
        r1[k] = load_raw8<DT>(a.x, at);
        r2[k] = load_raw8<DT>(a.x, at + D / 2);
      }
    }
  };
  fetch(h0);
#pragma unroll
  for (int k = 0; k < kItems; ++k) {
    const int item = k * team + me, i = item / kChunks, chunk = item % kChunks;
    if (!kv && i < n) load_cos_sin(a, z.p0 + i, chunk * 8, c[k], s[k]);
  }
  for (int h = h0; h < h0 + heads; ++h) {     // (every team of the CTA makes all turns: barriers)
    const bool some = n > 0 && h < h1;
    float* sc = some ? scale_at(a, kv, z.page, h) : nullptr;
    const float old = some && z.start > 0 ? *sc : 0.f;
    float x1[kItems][8], x2[kItems][8];
    float amax = 0.f;
#pragma unroll
    for (int k = 0; k < kItems; ++k)
      if (some && (k * team + me) / kChunks < n) {
        floats8<DT>(r1[k], x1[k]);
        floats8<DT>(r2[k], x2[k]);
        if (!kv) rotate8(x1[k], x2[k], c[k], s[k]);
        amax = max_abs(x1[k], x2[k], amax);
      }
    if (h + 1 < h1) fetch(h + 1);
    amax = warp_max(amax);
    float* slot = top[h & 1];                 // (a slot is written again two barriers later)
    if ((threadIdx.x & 31) == 0) slot[threadIdx.x / 32] = amax;
    __syncthreads();                          // (also: the old scale has been read before it is replaced)
    if (!some) continue;
    const int first = (threadIdx.x / team) * (team / 32);
    for (int i = 0; i < team / 32; ++i) amax = fmaxf(amax, slot[first + i]);
    const float scale = fmaxf(old, block_scale<INT8>(amax));
    uint8_t* data = block_at(a, kv, z.page, h);
    if (z.start > 0 && scale > old)
      for (int item = me; item < z.start * kChunks; item += team)
        rescale16<INT8>(data + (long)(item / kChunks) * a.c.token_stride + item % kChunks * 16, __fdiv_rn(old, scale));
    if (me == 0) *sc = scale;
    const float inv = __fdiv_rn(1.f, scale);
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int item = k * team + me, i = item / kChunks;
      if (i < n) store_codes<D, INT8>(data + (long)(z.start + i) * a.c.token_stride, item % kChunks, x1[k], x2[k], inv);
    }
  }
}

// Short units: one launch, the first CTAs store k and v, the others rotate q.
template <int DT, int D, bool INT8>
__global__ void __launch_bounds__(kThreads, 4) append_short_kernel(AppendArgs a, int store_ctas) {
  pdl_trigger();
  pdl_wait();
  if (int(blockIdx.x) < store_ctas) store_short<DT, D, INT8>(a, blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5));
  else rope_q<DT, D>(a, (blockIdx.x - store_ctas) * kThreads + threadIdx.x);
}

// Prompts: two launches, since the two want different shapes: k and v 128 registers a thread for what
// they hold and prefetch, q as many threads as there are. (16381 tokens: 80 us; one launch of both 88;
// k and v with 16 values a thread, twice the threads and 64 registers, 91.)
template <int DT, int D, bool INT8>
__global__ void __launch_bounds__(512, 1) append_block_kernel(AppendArgs a, int heads) {
  pdl_trigger();
  pdl_wait();
  store_block<DT, D, INT8>(a, blockIdx.x, heads);
}

template <int DT, int D>
__global__ void __launch_bounds__(kThreads, 4) rope_q_kernel(AppendArgs a) {
  pdl_trigger();
  pdl_wait();
  rope_q<DT, D>(a, blockIdx.x * kThreads + threadIdx.x);
}

template <int DT, int D, bool INT8>
cudaError_t launch_append(const AppendArgs& a, cudaStream_t s, int* launched) {
  const long items = (long)a.T * (D / 16) * ((a.H + kQHeads - 1) / kQHeads);
  const long q_ctas = (items + kThreads - 1) / kThreads;
  if (items + kThreads > 0x7fffffffl || (long)a.U * 2 * a.c.Hkv > 0x3fffffffl) return cudaErrorInvalidValue;
  // Whole blocks from 12 tokens a unit on average (entries that pad the list count): 64 rows of 8 heads and 128 dims take 10.2 us in short
  // units and 19.5 us in blocks at 1 token a row, 16.4 and 21.5 at 8, 26.6 and 23.6 at 16; 5 rows of
  // 2048 tokens 30.7 and 19.4.
  if ((long)a.T < 12l * a.U || a.U == 0) {
    const long warps = (long)a.U * 2 * a.c.Hkv, s_ctas = (warps + kThreads / 32 - 1) / (kThreads / 32);
    *launched = 1;
    return launch_pdl(append_short_kernel<DT, D, INT8>, dim3(unsigned(q_ctas + s_ctas)), dim3(kThreads), 0, s, a, int(s_ctas));
  }
  const int team = block_threads(a.c.P, D), threads = team > 256 ? team : 256, per = threads / team;
  // heads a team goes through: as many as leave four CTAs an SM
  int heads = 1;
  while (heads < a.c.Hkv && (long)a.U * 2 * (a.c.Hkv / (2 * heads)) >= 4l * a.num_sms * per) heads *= 2;
  const long teams = (long)a.U * 2 * ((a.c.Hkv + heads - 1) / heads);
  cudaError_t e = launch_pdl(append_block_kernel<DT, D, INT8>, dim3(unsigned((teams + per - 1) / per)), dim3(threads), 0, s, a, heads);
  if (e != cudaSuccess) return e;
  *launched = 2;
  return launch_pdl(rope_q_kernel<DT, D>, dim3(unsigned(q_ctas)), dim3(kThreads), 0, s, a);
}

template <int DT, int D>
cudaError_t append_code(const AppendArgs& a, cudaStream_t s, int* launched) {
  return a.c.code == kInt8 ? launch_append<DT, D, true>(a, s, launched) : launch_append<DT, D, false>(a, s, launched);
}

template <int DT>
cudaError_t append_dim(const AppendArgs& a, cudaStream_t s, int* launched) {
  return a.c.D == 64 ? append_code<DT, 64>(a, s, launched) : append_code<DT, 128>(a, s, launched);
}

// 16 codes of one (row, head) a thread.
template <int D, bool INT8>
__global__ void __launch_bounds__(kThreads) gather_kernel(GatherArgs a) {
  constexpr int kChunks = D / 16;
  pdl_trigger();
  pdl_wait();
  const int h = blockIdx.y, kv = blockIdx.z;
  const int item = blockIdx.x * kThreads + threadIdx.x;
  const int i = item / kChunks, chunk = item % kChunks;
  if (i >= a.n) return;
  const int page = a.table[i / a.c.P];
  uint4 v = make_uint4(0, 0, 0, 0);
  float scale = 0.f;
  if (page >= 0 && page < a.c.pages) {
    v = ld_nc_v4((kv ? a.c.v : a.c.k) + (long)page * a.c.page_stride + (long)h * a.c.head_stride +
                 (long)(i % a.c.P) * a.c.token_stride + chunk * 16);
    scale = (kv ? a.c.v_scale : a.c.k_scale)[(long)page * a.c.scale_page_stride + (long)h * a.c.scale_head_stride];
  }
  const uint32_t in[4] = {v.x, v.y, v.z, v.w};
  uint32_t out[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t lo, hi;
    decode4<INT8>(in[j], lo, hi);
    const float2 x = half2_floats(lo), y = half2_floats(hi);
    out[2 * j] = pack_bf16x2(x.x * scale, x.y * scale);
    out[2 * j + 1] = pack_bf16x2(y.x * scale, y.y * scale);
  }
  uint4* o = reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(kv ? a.v_out : a.k_out) +
                                      (long)h * a.out_head_stride + (long)i * D + chunk * 16);
  o[0] = make_uint4(out[0], out[1], out[2], out[3]);
  o[1] = make_uint4(out[4], out[5], out[6], out[7]);
}

template <int D, bool INT8>
cudaError_t launch_gather(const GatherArgs& a, cudaStream_t s) {
  const long items = (long)a.n * (D / 16);
  const dim3 grid(unsigned((items + kThreads - 1) / kThreads), unsigned(a.c.Hkv), 2);
  return launch_pdl(gather_kernel<D, INT8>, grid, dim3(kThreads), 0, s, a);
}

const char* check_cache(const Cache& c) {
  if (c.D != 64 && c.D != 128) return "8-bit cache: head_dim must be 64 or 128";
  if (c.P != 16 && c.P != 32 && c.P != 64 && c.P != 128) return "8-bit cache: page must be 16, 32, 64 or 128 tokens";
  if (c.pages < 1 || c.Hkv < 1) return "8-bit cache: no pages or heads";
  if (c.page_stride % 16 || c.head_stride % 16 || c.token_stride % 16 || reinterpret_cast<uintptr_t>(c.k) % 16 ||
      reinterpret_cast<uintptr_t>(c.v) % 16)
    return "8-bit cache: rows must start on 16-byte boundaries";
  return nullptr;
}

}  // namespace

const char* rope_append(const AppendArgs& a, cudaStream_t s, int* launched) {
  *launched = 0;
  if (const char* e = check_cache(a.c)) return e;
  if (a.T < 1) return nullptr;
  if (a.row_stride % 8 || reinterpret_cast<uintptr_t>(a.x) % 16 || reinterpret_cast<uintptr_t>(a.q_out) % 16)
    return "rope_append_kv8: rows must start on 16-byte boundaries";
  cudaError_t e = a.dtype == kF32    ? append_dim<kF32>(a, s, launched)
                  : a.dtype == kBF16 ? append_dim<kBF16>(a, s, launched)
                                     : append_dim<kF16>(a, s, launched);
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

const char* gather(const GatherArgs& a, cudaStream_t s) {
  if (const char* e = check_cache(a.c)) return e;
  if (a.n < 1) return nullptr;
  if ((a.n + a.c.P - 1) / a.c.P > a.width) return "gather_kv8: more rows than the table holds";
  if (a.c.Hkv > 65535) return "gather_kv8: too many heads";
  if ((long)a.n * (a.c.D / 16) >= (1l << 31) - kThreads) return "gather_kv8: too many rows";   // (32-bit piece numbers)
  cudaError_t e = a.c.D == 64 ? (a.c.code == kInt8 ? launch_gather<64, true>(a, s) : launch_gather<64, false>(a, s))
                              : (a.c.code == kInt8 ? launch_gather<128, true>(a, s) : launch_gather<128, false>(a, s));
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace kv8
}  // namespace hcp
