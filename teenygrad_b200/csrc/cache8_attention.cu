// Causal attention over the 8-bit key/value cache (layout in teeny_cache8.h).
#include "common.cuh"
#include "kernels.h"
#include "mma.cuh"

namespace teeny {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float load_one(const bf16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load_one(const float* p) { return *p; }
__device__ __forceinline__ void store_one(bf16* p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void store_one(float* p, float x) { *p = x; }
__device__ __forceinline__ float4 decode4(uint32_t w) {
  const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xffffu), __NV_E4M3);
  const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ float capped(float s, float softcap) { return softcap > 0.0f ? softcap * tanhf(s / softcap) : s; }

// One CTA of four warps for a (row, query head); warp w takes the keys w, w + 4, .., lane l the dimensions 4l .. 4l + 3.
template <typename T>
__global__ void __launch_bounds__(128) cache8_rows_kernel(const Cache8 c, const Cache8Attn a, const SeqDesc* seqs, int max_len, float* lse_out) {
  __shared__ float sm_m[4], sm_l[4], sm_o[4][kCache8Head];
  pdl_wait();
  const SeqDesc sq = seqs[blockIdx.y];
  const int i = blockIdx.x / a.Hq, h = blockIdx.x % a.Hq, hk = h / (a.Hq / c.H);
  if (!cache8_fits(sq, c, a.rows, max_len) || i >= sq.len) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, live = sq.pos + i + 1;
  const size_t row = sq.row0 + i, head = static_cast<size_t>(sq.slot) * c.H + hk;
  float q[4], o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int e = 0; e < 4; ++e) q[e] = 4 * lane < c.D ? load_one(static_cast<const T*>(a.q) + row * a.ldq + h * c.D + 4 * lane + e) : 0.0f;
  for (int j = warp; j < live; j += 4) {
    float s = 0.0f;
    if (4 * lane < c.D) {
      const float4 x = decode4(*reinterpret_cast<const uint32_t*>(c.k + (head * c.cap + j) * c.D + 4 * lane));
      s = q[0] * x.x + q[1] * x.y + q[2] * x.z + q[3] * x.w;
    }
    s = capped(warp_sum(s) * c.ks[head * c.blocks + j / c.B] * a.scale, a.softcap);
    const float top = fmaxf(m, s), old = m == -INFINITY ? 0.0f : expf(m - top), p = expf(s - top);
    m = top;
    l = l * old + p;
    if (4 * lane < c.V) {
      const float4 x = decode4(*reinterpret_cast<const uint32_t*>(c.v + (head * c.cap + j) * c.V + 4 * lane));
      const float pv = p * c.vs[head * c.blocks + j / c.B];
      o[0] = o[0] * old + pv * x.x; o[1] = o[1] * old + pv * x.y; o[2] = o[2] * old + pv * x.z; o[3] = o[3] * old + pv * x.w;
    }
  }
  if (lane == 0) { sm_m[warp] = m; sm_l[warp] = l; }
#pragma unroll
  for (int e = 0; e < 4; ++e) sm_o[warp][4 * lane + e] = o[e];
  __syncthreads();
  float top = fmaxf(fmaxf(sm_m[0], sm_m[1]), fmaxf(sm_m[2], sm_m[3])), sum = 0.0f, x = 0.0f;
  const int d = threadIdx.x;
  for (int w = 0; w < 4; ++w) {
    const float f = sm_m[w] == -INFINITY ? 0.0f : expf(sm_m[w] - top);
    sum += sm_l[w] * f;
    x += sm_o[w][d] * f;
  }
  if (a.sink) sum += expf(a.sink[h] - top);
  if (lse_out && d == 0) lse_out[row * a.Hq + h] = top + logf(sum);
  if (d >= c.V) return;
  x /= sum;
  if (a.gate) x *= sigmoid_f(load_one(static_cast<const T*>(a.gate) + row * a.ldg + h * c.V + d));
  store_one(static_cast<T*>(a.out) + row * a.ldo + h * c.V + d, x);
}

// A warp for a (key, kv head): the probabilities that the entry's rows gave it, from the rows' lse.
template <typename T>
__global__ void __launch_bounds__(128) cache8_weights_kernel(const Cache8 c, const Cache8Attn a, const SeqDesc* seqs, int max_len, const float* lse) {
  pdl_wait();
  const SeqDesc sq = seqs[blockIdx.z];
  if (!cache8_fits(sq, c, a.rows, max_len)) return;
  const int hk = blockIdx.y, lane = threadIdx.x & 31, group = a.Hq / c.H;
  for (int j = blockIdx.x * 4 + (threadIdx.x >> 5); j < sq.pos + sq.len; j += gridDim.x * 4) {
    const size_t head = static_cast<size_t>(sq.slot) * c.H + hk;
    float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (4 * lane < c.D) x = decode4(*reinterpret_cast<const uint32_t*>(c.k + (head * c.cap + j) * c.D + 4 * lane));
    const float scale = c.ks[head * c.blocks + j / c.B] * a.scale;
    float sum = 0.0f;
    for (int i = max(0, j - sq.pos); i < sq.len; ++i)
      for (int g = 0; g < group; ++g) {
        const size_t row = sq.row0 + i;
        const T* q = static_cast<const T*>(a.q) + row * a.ldq + (hk * group + g) * c.D + 4 * lane;
        float s = 0.0f;
        if (4 * lane < c.D) s = load_one(q) * x.x + load_one(q + 1) * x.y + load_one(q + 2) * x.z + load_one(q + 3) * x.w;
        sum += expf(capped(warp_sum(s) * scale, a.softcap) - lse[row * a.Hq + hk * group + g]);
      }
    float* w = c.w + head * c.cap + j;
    if (lane == 0) *w = a.decay == 0.0f ? sum : a.decay * *w + sum;
  }
}

}  // namespace

size_t cache8_attention_scratch_bytes(const Cache8&, int, int Hq, int rows, int, int, bool weights) {
  return weights ? static_cast<size_t>(rows) * Hq * 4 : 0;
}

int cache8_attention(const Cache8& c, const Cache8Attn& a, const SeqDesc* seqs, const SeqDesc*, int n_seqs, int max_len, cudaStream_t st) {
  float* lse = a.lse ? a.lse : a.weights ? static_cast<float*>(a.scratch) : nullptr;
  const dim3 grid(static_cast<unsigned>(max_len) * a.Hq, n_seqs);
  if (a.f32) launch_kernel(cache8_rows_kernel<float>, grid, dim3(128), 0, st, 1, c, a, seqs, max_len, lse);
  else launch_kernel(cache8_rows_kernel<bf16>, grid, dim3(128), 0, st, 1, c, a, seqs, max_len, lse);
  if (a.weights) {
    const dim3 wgrid(512, c.H, n_seqs);
    if (a.f32) launch_kernel(cache8_weights_kernel<float>, wgrid, dim3(128), 0, st, 1, c, a, seqs, max_len, static_cast<const float*>(lse));
    else launch_kernel(cache8_weights_kernel<bf16>, wgrid, dim3(128), 0, st, 1, c, a, seqs, max_len, static_cast<const float*>(lse));
  }
  return static_cast<int>(cudaGetLastError());
}

}  // namespace teeny
