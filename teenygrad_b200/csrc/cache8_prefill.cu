// Prompts and long portions over the 8-bit cache: their work is the products, not the cache's bytes, so an entry's live tokens are widened to bf16 in
// scratch once (exact: an E4M3 number times a power of two) and the tcgen05 kernel of attention_prefill.cu runs on those.  Widening
// reads one byte and writes two for each number, 0.8 KB a token and kv head at head size 128, against len * group * 512 multiply-adds.
#include "common.cuh"
#include "kernels.h"

namespace teeny {

namespace {

constexpr int kTile = 128;       // tokens of a widening CTA, and the attention kernel's key tile: an entry's region ends at a multiple
constexpr int kBudget = 65536;   // tokens whose widened form is held at a time (or one slot's, if that is more)
constexpr int kMostEntries = 128;

struct Widened {
  bf16 *k, *v;   // [kv heads][n_seqs * key_rows][dim]
  int* nan;      // [n_seqs][kv heads][tiles]: a new token's value holds a NaN
  int n_seqs, key_rows, tiles;
};

// 16 codes times a scale
__device__ __forceinline__ void widen16(const uint4& w, float scale, uint4 (&out)[2]) {
  const uint32_t r[4] = {w.x, w.y, w.z, w.w};
  uint32_t o[8];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const __half2_raw x = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(r[i] >> (16 * h) & 0xffffu), __NV_E4M3);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x));
      o[2 * i + h] = pack_bf16x2(f.x * scale, f.y * scale);
    }
  out[0] = make_uint4(o[0], o[1], o[2], o[3]);
  out[1] = make_uint4(o[4], o[5], o[6], o[7]);
}

// blockIdx = (tile of 128 tokens, 2 * head + (values), entry).  Behind the live tokens, to the tile's end, zeros.  NaN values of tokens that not all of the
// entry's rows see become zeros as well (a masked probability of zero times NaN is NaN) and are noted.
__global__ void __launch_bounds__(256) cache8_widen_kernel(const Cache8 c, const Widened to, const SeqDesc* seqs, int min_len, int max_len, int rows) {
  pdl_wait();
  const SeqDesc sq = seqs[blockIdx.z];
  if (sq.len < min_len || !cache8_fits(sq, c, rows, max_len)) return;
  const int live = sq.pos + sq.len, t0 = blockIdx.x * kTile;
  if (t0 >= live) return;
  const int head = blockIdx.y >> 1, of_v = blockIdx.y & 1, d = of_v ? c.V : c.D, per = d / 16;
  const size_t row = static_cast<size_t>(sq.slot) * c.H + head;
  const uint4* src = reinterpret_cast<const uint4*>((of_v ? c.v : c.k) + (row * c.cap + t0) * d);
  const float* scales = (of_v ? c.vs : c.ks) + row * c.blocks;
  uint4* dst = reinterpret_cast<uint4*>((of_v ? to.v : to.k) + (static_cast<size_t>(head) * to.n_seqs * to.key_rows + static_cast<size_t>(blockIdx.z) * to.key_rows + t0) * d);
  bool nan = false;
  const int chunks = kTile * per;
#pragma unroll 4
  for (int i = threadIdx.x; i < chunks; i += 256) {
    const int t = t0 + i / per;
    uint4 w = make_uint4(0u, 0u, 0u, 0u);
    float scale = 0.0f;
    if (t < live) {
      w = src[i];
      scale = scales[t / c.B];
    }
    if (of_v && t >= sq.pos) {
      uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t is = ((word[k] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;  // bytes 0x7f, 0xff
        if (is) {
          nan = true;
          word[k] &= ~((is >> 7) * 0xffu);
        }
      }
      w = make_uint4(word[0], word[1], word[2], word[3]);
    }
    uint4 o[2];
    widen16(w, scale, o);
    dst[2 * i] = o[0];
    dst[2 * i + 1] = o[1];
  }
  if (of_v) {
    const int any = __syncthreads_or(nan);
    if (threadIdx.x == 0) to.nan[(static_cast<size_t>(blockIdx.z) * c.H + head) * to.tiles + blockIdx.x] = any;
  }
}

// Puts the NaN values back: column d of an output row is NaN from the first token on whose value is NaN there.  blockIdx = (head, entry).
__global__ void __launch_bounds__(128) cache8_nan_kernel(const Cache8 c, const Cache8Attn a, const Widened w, const SeqDesc* seqs, int min_len, int max_len) {
  pdl_wait();
  const SeqDesc sq = seqs[blockIdx.y];
  if (sq.len < min_len || !cache8_fits(sq, c, a.rows, max_len)) return;
  const int live = sq.pos + sq.len, head = blockIdx.x;
  const int* flags = w.nan + (static_cast<size_t>(blockIdx.y) * c.H + head) * w.tiles;
  int any = 0;
  for (int t = sq.pos / kTile + threadIdx.x; t * kTile < live; t += 128) any |= flags[t];
  if (!__syncthreads_or(any)) return;
  const int d = threadIdx.x, G = a.Hq / c.H;
  if (d >= c.V) return;
  const uint8_t* v = c.v + ((static_cast<size_t>(sq.slot) * c.H + head) * c.cap) * c.V + d;
  int first = sq.pos;
  while (first < live && (v[static_cast<size_t>(first) * c.V] & 0x7f) != 0x7f) ++first;
  for (int i = first - sq.pos; i < sq.len; ++i)
    for (int g = 0; g < G; ++g)
      static_cast<bf16*>(a.out)[(static_cast<size_t>(sq.row0) + i) * a.ldo + static_cast<size_t>(head * G + g) * c.V + d] = __ushort_as_bfloat16(0x7fff);
}

Widened widened_of(const Cache8& c, int n_seqs, void* scratch, size_t* bytes) {
  Widened w{};
  w.key_rows = (c.cap + kTile - 1) / kTile * kTile;
  w.tiles = w.key_rows / kTile;
  const int at_once = kBudget / w.key_rows < 1 ? 1 : kBudget / w.key_rows < kMostEntries ? kBudget / w.key_rows : kMostEntries;
  w.n_seqs = n_seqs < at_once ? n_seqs : at_once;
  const size_t rows = static_cast<size_t>(c.H) * w.n_seqs * w.key_rows;
  uint8_t* p = static_cast<uint8_t*>(scratch);
  w.k = reinterpret_cast<bf16*>(p);
  w.v = reinterpret_cast<bf16*>(p + rows * c.D * 2);
  w.nan = reinterpret_cast<int*>(p + rows * (c.D + c.V) * 2);
  *bytes = rows * (c.D + c.V) * 2 + (static_cast<size_t>(w.n_seqs) * c.H * w.tiles * 4 + 255) / 256 * 256;
  return w;
}

}  // namespace

int cache8_prefill_min_len(const Cache8& c, int Hq) {
  const int G = Hq / c.H, n = 192 / G;
  return n < 32 ? 32 : n;
}
bool cache8_prefill_takes(const Cache8& c, const Cache8Attn& a, int max_len) {
  const uintptr_t bases = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.out) | reinterpret_cast<uintptr_t>(a.gate);
  return !a.f32 && max_len >= cache8_prefill_min_len(c, a.Hq) && (bases & 15) == 0 && ((a.ldq | a.ldo | a.ldg) & 7) == 0 && a.scale > 0.0f &&
         a.scale < 1e30f;
}
size_t cache8_prefill_scratch_bytes(const Cache8& c, int n_seqs) {
  size_t n;
  widened_of(c, n_seqs, nullptr, &n);
  return n;
}
int cache8_prefill(const Cache8& c, const Cache8Attn& a, float* lse2, void* scratch, const SeqDesc* seqs, int n_seqs, int max_len, cudaStream_t st) {
  size_t bytes;
  Widened w = widened_of(c, n_seqs, scratch, &bytes);
  const int min_len = cache8_prefill_min_len(c, a.Hq), at_once = w.n_seqs;
  for (int e = 0; e < n_seqs; e += at_once) {
    w.n_seqs = n_seqs - e < at_once ? n_seqs - e : at_once;
    launch_kernel(cache8_widen_kernel, dim3(w.tiles, 2 * c.H, w.n_seqs), dim3(256), 0, st, 1, c, w, seqs + e, min_len, max_len, a.rows);
    const bool pdl = pdl_enabled();
    pdl_set_enabled(true);
    const int rc = attention_prefill_ragged(c, a, w.k, w.v, w.key_rows, lse2, seqs + e, w.n_seqs, min_len, max_len, st);
    if (rc == 0) launch_kernel(cache8_nan_kernel, dim3(c.H, w.n_seqs), dim3(128), 0, st, 1, c, a, w, seqs + e, min_len, max_len);
    pdl_set_enabled(pdl);
    if (rc) return rc;
  }
  return static_cast<int>(cudaGetLastError());
}

}  // namespace teeny
