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
// Both are bound by memory traffic.
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

// q of one (token, 8-element chunk) for every head of a group.
constexpr int kQHeads = 8;

template <int DT, int D>
__device__ __forceinline__ void rope_q(const AppendArgs& a, long item) {
  constexpr int kChunks = D / 16;
  const int chunk = int(item % kChunks);
  const long rest = item / kChunks;
  const int groups = (a.H + kQHeads - 1) / kQHeads;
  const int t = int(rest / groups), h0 = int(rest % groups) * kQHeads;
  if (t >= a.T) return;
  const int pos = a.pos[t];
  float c[8], s[8];
  const bool ok = pos >= 0 && pos < a.max_pos;
  if (!ok && chunk == 0 && h0 == 0) report_error(a.status, int(StatusCode::kOutOfBounds), 401, pos, t);
  load_cos_sin(a, ok ? pos : 0, chunk * 8, c, s);
  const int h1 = min(a.H, h0 + kQHeads);
#pragma unroll 4
  for (int h = h0; h < h1; ++h) {
    float x1[8], x2[8];
    const long at = (long)t * a.row_stride + (long)h * D + chunk * 8;
    load8<DT>(a.x, at, x1);
    load8<DT>(a.x, at + D / 2, x2);
    rotate8(x1, x2, c, s);
    uint4* o = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.q_out) + ((long)t * a.H + h) * D + chunk * 8);
    o[0] = make_uint4(pack16(a.q_dtype, x1[0], x1[1]), pack16(a.q_dtype, x1[2], x1[3]),
                      pack16(a.q_dtype, x1[4], x1[5]), pack16(a.q_dtype, x1[6], x1[7]));
    o[D / 16] = make_uint4(pack16(a.q_dtype, x2[0], x2[1]), pack16(a.q_dtype, x2[2], x2[3]),
                           pack16(a.q_dtype, x2[4], x2[5]), pack16(a.q_dtype, x2[6], x2[7]));
  }
}

// One warp per (unit, KV head, k or v): the maximum over the unit's tokens, the scale, the codes.
template <int DT, int D, bool INT8>
__device__ __forceinline__ void store_unit(const AppendArgs& a, long w) {
  constexpr int kChunks = D / 16, kTok = 32 / kChunks;  // tokens a warp covers at a time
  const int lane = threadIdx.x & 31;
  const int kv = int(w & 1);
  const long rest = w >> 1;
  const int h = int(rest % a.c.Hkv);
  const long ui = rest / a.c.Hkv;
  if (ui >= a.U) return;
  const int4 u = a.unit[ui];
  const int row = u.x, t0 = u.y, n = u.z, p0 = u.w;
  if (row < 0) return;
  const int P = a.c.P;
  const int block = p0 / P, start = p0 - block * P;
  const bool ok = row < a.R && t0 >= 0 && n >= 1 && t0 + n <= a.T && p0 >= 0 && start + n <= P && block < a.width;
  const int page = ok ? a.table[(long)row * a.width + block] : -1;
  if (page < 0 || page >= a.c.pages) {
    if (lane == 0) report_error(a.status, int(StatusCode::kOutOfBounds), 402, page, int(ui));
    return;
  }
  const int chunk = lane % kChunks, sub = lane / kChunks;
  const int col = a.H + (kv ? a.c.Hkv : 0) + h;
  auto row_values = [&](int i, float (&x1)[8], float (&x2)[8]) {
    const long at = (long)(t0 + i) * a.row_stride + (long)col * D + chunk * 8;
    load8<DT>(a.x, at, x1);
    load8<DT>(a.x, at + D / 2, x2);
    if (!kv) {
      float c[8], s[8];
      load_cos_sin(a, min(p0 + i, a.max_pos - 1), chunk * 8, c, s);
      rotate8(x1, x2, c, s);
    }
  };
  float amax = 0.f;
  for (int i = sub; i < n; i += kTok) {
    float x1[8], x2[8];
    row_values(i, x1, x2);
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = fmaxf(amax, fmaxf(fabsf(x1[j]), fabsf(x2[j])));
  }
  amax = warp_max(amax);
  float* scale_at = (kv ? a.c.v_scale : a.c.k_scale) + (long)page * a.c.scale_page_stride + (long)h * a.c.scale_head_stride;
  const float old = start > 0 ? *scale_at : 0.f;
  const float scale = fmaxf(old, block_scale<INT8>(amax));
  __syncwarp();
  uint8_t* data = (kv ? a.c.v : a.c.k) + (long)page * a.c.page_stride + (long)h * a.c.head_stride;
  if (start > 0 && scale > old) {
    const float f = __fdiv_rn(old, scale);
    for (int i = sub; i < start; i += kTok) {
      uint4* p = reinterpret_cast<uint4*>(data + (long)i * a.c.token_stride + chunk * 16);
      const uint4 v = *p;
      uint32_t in[4] = {v.x, v.y, v.z, v.w}, out[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t lo, hi;
        decode4<INT8>(in[j], lo, hi);
        const float2 x = half2_floats(lo), y = half2_floats(hi);
        out[j] = encode4<INT8>(x.x * f, x.y * f, y.x * f, y.y * f);
      }
      *p = make_uint4(out[0], out[1], out[2], out[3]);
    }
  }
  if (lane == 0) *scale_at = scale;
  const float inv = __fdiv_rn(1.f, scale);  // exact: a power of two (an old scale may be another value)
  for (int i = sub; i < n; i += kTok) {
    float x1[8], x2[8];
    row_values(i, x1, x2);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x1[j] *= inv;
      x2[j] *= inv;
    }
    uint8_t* p = data + (long)(start + i) * a.c.token_stride + chunk * 8;
    *reinterpret_cast<uint2*>(p) = make_uint2(encode4<INT8>(x1[0], x1[1], x1[2], x1[3]),
                                              encode4<INT8>(x1[4], x1[5], x1[6], x1[7]));
    *reinterpret_cast<uint2*>(p + D / 2) = make_uint2(encode4<INT8>(x2[0], x2[1], x2[2], x2[3]),
                                                      encode4<INT8>(x2[4], x2[5], x2[6], x2[7]));
  }
}

template <int DT, int D, bool INT8>
__global__ void __launch_bounds__(kThreads) append_kernel(AppendArgs a, int q_ctas) {
  pdl_trigger();
  pdl_wait();
  if (int(blockIdx.x) < q_ctas) {
    rope_q<DT, D>(a, (long)blockIdx.x * kThreads + threadIdx.x);
  } else {
    store_unit<DT, D, INT8>(a, ((long)blockIdx.x - q_ctas) * (kThreads / 32) + (threadIdx.x >> 5));
  }
}

template <int DT, int D, bool INT8>
cudaError_t launch_append(const AppendArgs& a, cudaStream_t s) {
  const long items = (long)a.T * (D / 16) * ((a.H + kQHeads - 1) / kQHeads);
  const long q_ctas = (items + kThreads - 1) / kThreads;
  const long warps = (long)a.U * a.c.Hkv * 2;
  const long s_ctas = (warps + kThreads / 32 - 1) / (kThreads / 32);
  if (q_ctas + s_ctas > 0x7fffffffl) return cudaErrorInvalidValue;
  return launch_pdl(append_kernel<DT, D, INT8>, dim3(unsigned(q_ctas + s_ctas)), dim3(kThreads), 0, s, a, int(q_ctas));
}

template <int DT, int D>
cudaError_t append_code(const AppendArgs& a, cudaStream_t s) {
  return a.c.code == kInt8 ? launch_append<DT, D, true>(a, s) : launch_append<DT, D, false>(a, s);
}

template <int DT>
cudaError_t append_dim(const AppendArgs& a, cudaStream_t s) {
  return a.c.D == 64 ? append_code<DT, 64>(a, s) : append_code<DT, 128>(a, s);
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

const char* rope_append(const AppendArgs& a, cudaStream_t s) {
  if (const char* e = check_cache(a.c)) return e;
  if (a.T < 1 || a.U < 1) return nullptr;
  if (a.row_stride % 8 || reinterpret_cast<uintptr_t>(a.x) % 16 || reinterpret_cast<uintptr_t>(a.q_out) % 16)
    return "rope_append_kv8: rows must start on 16-byte boundaries";
  cudaError_t e = a.dtype == kF32 ? append_dim<kF32>(a, s) : a.dtype == kBF16 ? append_dim<kBF16>(a, s) : append_dim<kF16>(a, s);
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

const char* gather(const GatherArgs& a, cudaStream_t s) {
  if (const char* e = check_cache(a.c)) return e;
  if (a.n < 1) return nullptr;
  if ((a.n + a.c.P - 1) / a.c.P > a.width) return "gather_kv8: more rows than the table holds";
  if (a.c.Hkv > 65535) return "gather_kv8: too many heads";
  cudaError_t e = a.c.D == 64 ? (a.c.code == kInt8 ? launch_gather<64, true>(a, s) : launch_gather<64, false>(a, s))
                              : (a.c.code == kInt8 ? launch_gather<128, true>(a, s) : launch_gather<128, false>(a, s));
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace kv8
}  // namespace hcp
