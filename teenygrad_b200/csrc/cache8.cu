// The 8-bit key/value cache: appending tokens, evicting them, and the entry points of teeny_cache8.h.
//
// Scales are powers of two, so that holding a code at another scale is a shift of its exponent, exact unless the result leaves E4M3's
// normal range.  A block's scale is 2^k with the smallest k >= -126 for which its largest number is at most 448 * 2^k.
#include <algorithm>
#include <cstdlib>

#include "../../include/teeny_cache8.h"
#include "common.cuh"
#include "kernels.h"

namespace teeny {

namespace {

constexpr int kThreads = 256;

// Exponent of the scale for numbers up to amax (finite, >= 0): 448 = 1.75 * 2^8.
__device__ __forceinline__ int scale_exponent(float amax) {
  const unsigned u = __float_as_uint(amax);
  return max(-126, static_cast<int>(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0));
}
__device__ __forceinline__ float pow2(int k) { return __uint_as_float(static_cast<unsigned>(k + 127) << 23); }  // -126 <= k <= 127
__device__ __forceinline__ int exponent_of(float scale) { return static_cast<int>(__float_as_uint(scale) >> 23) - 127; }

// 16 codes times 2^j: in f16 the products are exact down to 2^-24, far below the least code.
__device__ __forceinline__ uint4 rescale16(uint4 v, int j) {
  if (j == 0) return v;
  uint32_t r[4] = {v.x, v.y, v.z, v.w};
  const bool far = j > 14;  // (a code can grow by up to 2^17: two factors)
  const __half2 f0 = __float2half2_rn(pow2(max(-24, min(j, 14)))), f1 = __float2half2_rn(pow2(far ? min(j - 14, 14) : 0));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t out[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const __half2_raw x = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(r[i] >> (16 * h) & 0xffffu), __NV_E4M3);
      __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&x), f0);
      if (far) y = __hmul2(y, f1);
      out[h] = __nv_cvt_halfraw2_to_fp8x2(*reinterpret_cast<const __half2_raw*>(&y), __NV_SATFINITE, __NV_E4M3);
    }
    r[i] = __byte_perm(out[0], out[1], 0x5410);
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}
// Largest magnitude of 16 codes, NaN left out
__device__ __forceinline__ float top_of(const uint4& v) {
  const uint32_t r[4] = {v.x, v.y, v.z, v.w};
  __half2 top = __float2half2_rn(0.0f);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const __half2_raw x = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(r[i >> 1] >> (16 * (i & 1)) & 0xffffu), __NV_E4M3);
    top = __hmax2(top, __habs2(*reinterpret_cast<const __half2*>(&x)));
  }
  return fmaxf(__low2float(top), __high2float(top));
}

// 16 numbers of a row as they are in memory (vec: in 16-byte pieces), their largest magnitude, and their codes
template <typename T>
struct Sixteen;
template <>
struct Sixteen<bf16> {
  uint32_t w[8];
  __device__ __forceinline__ void load(const bf16* p, bool vec) {
    if (vec) {
      const uint4 a = reinterpret_cast<const uint4*>(p)[0], b = reinterpret_cast<const uint4*>(p)[1];
      w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = b.x; w[5] = b.y; w[6] = b.z; w[7] = b.w;
    } else {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = h[2 * i] | static_cast<uint32_t>(h[2 * i + 1]) << 16;
    }
  }
  __device__ __forceinline__ float top() const {  // (of a NaN and a number the number)
    __nv_bfloat162 m = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[0]));
#pragma unroll
    for (int i = 1; i < 8; ++i) m = __hmax2(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[i])));
    return fmaxf(__low2float(m), __high2float(m));
  }
  __device__ __forceinline__ float2 two(int i) const { return make_float2(bf16_lo(w[i]), bf16_hi(w[i])); }
};
template <>
struct Sixteen<float> {
  float2 x[8];
  __device__ __forceinline__ void load(const float* p, bool vec) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (vec) {
        const float4 v = reinterpret_cast<const float4*>(p)[i];
        x[2 * i] = make_float2(v.x, v.y);
        x[2 * i + 1] = make_float2(v.z, v.w);
      } else {
        x[2 * i] = make_float2(p[4 * i], p[4 * i + 1]);
        x[2 * i + 1] = make_float2(p[4 * i + 2], p[4 * i + 3]);
      }
    }
  }
  __device__ __forceinline__ float top() const {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, fmaxf(fabsf(x[i].x), fabsf(x[i].y)));
    return m;
  }
  __device__ __forceinline__ float2 two(int i) const { return x[i]; }
};
template <typename T>
__device__ __forceinline__ float top_finite(const Sixteen<T>& x) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = fabsf(x.two(i).x), b = fabsf(x.two(i).y);
    m = fmaxf(m, fmaxf(a < INFINITY ? a : 0.0f, b < INFINITY ? b : 0.0f));
  }
  return m;
}
// none of them beyond 448 after scaling (round to nearest even); infinite: some are not finite, and become NaN
template <typename T>
__device__ __forceinline__ uint4 encode16(const Sixteen<T>& x, float inv, bool infinite) {
  uint32_t r[4];
  const float2 f = make_float2(inv, inv);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t out = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float2 y = __fmul2_rn(x.two(2 * i + h), f);
      if (infinite) {
        if (!(fabsf(y.x) < INFINITY)) y.x = __uint_as_float(0x7fffffffu);
        if (!(fabsf(y.y) < INFINITY)) y.y = __uint_as_float(0x7fffffffu);
      }
      out |= static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(y, __NV_SATFINITE, __NV_E4M3)) << (16 * h);
    }
    r[i] = out;
  }
  return make_uint4(r[0], r[1], r[2], r[3]);
}
__device__ __forceinline__ float block_max(float v, float* sh) {
  v = warp_max(v);
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  float m = sh[0];
  for (int w = 1; w < static_cast<int>(blockDim.x >> 5); ++w) m = fmaxf(m, sh[w]);
  __syncthreads();
  return m;
}

// One CTA for the new tokens of one entry in one block of the cache: blockIdx = (block counted from the entry's first, 2 * head + (values), entry).
// A thread holds the 16-element pieces that it reads (up to NCH) until the scale is known: each number is read once.  Bound by HBM for prompts (16 of
// up to 2048 tokens, eight heads of 128, 130 MB: 23.3 us, 5.6 TB/s), by a launch's latency for single tokens (64 of them: 3.0 us).
template <typename T, int NCH>
__global__ void __launch_bounds__(kThreads) cache8_append_kernel(const Cache8 c, const Cache8Append a, const SeqDesc* seqs, int max_len, int vec) {
  __shared__ float sh[kThreads / 32];
  pdl_wait();
  const SeqDesc sq = seqs[blockIdx.z];
  if (!cache8_fits(sq, c, a.rows, max_len)) return;
  const int head = blockIdx.y >> 1, of_v = blockIdx.y & 1, d = of_v ? c.V : c.D, per = d / 16, step = blockDim.x;
  const int b = (sq.pos >> c.shift) + blockIdx.x, begin = max(sq.pos, b * c.B), end = min(sq.pos + sq.len, (b + 1) * c.B);
  if (begin >= end) return;
  const size_t row = static_cast<size_t>(sq.slot) * c.H + head;
  uint8_t* codes = (of_v ? c.v : c.k) + row * c.cap * d;
  float* scales = (of_v ? c.vs : c.ks) + row * c.blocks;
  const long long ld = of_v ? a.ldv : a.ldk;
  const T* src = static_cast<const T*>(of_v ? a.v : a.k) + (sq.row0 + begin - sq.pos) * ld + head * d;
  const bool older = begin > b * c.B;
  const float was = older ? scales[b] : 0.0f;
  const int chunks = (end - begin) * per;
  Sixteen<T> x[NCH];
  float amax = 0.0f;
#pragma unroll
  for (int m = 0; m < NCH; ++m) {
    const int i = threadIdx.x + m * step;
    if (i < chunks) {
      const int t = per == 8 ? i >> 3 : i / per;
      x[m].load(src + t * ld + (i - t * per) * 16, vec);
    }
  }
#pragma unroll
  for (int m = 0; m < NCH; ++m)
    if (threadIdx.x + m * step < chunks) amax = fmaxf(amax, x[m].top());
  amax = block_max(amax, sh);
  const bool infinite = amax == INFINITY;
  if (infinite) {  // (the same for the CTA)
    amax = 0.0f;
#pragma unroll
    for (int m = 0; m < NCH; ++m)
      if (threadIdx.x + m * step < chunks) amax = fmaxf(amax, top_finite(x[m]));
    amax = block_max(amax, sh);
  }
  const float fresh = pow2(scale_exponent(amax)), scale = older ? fmaxf(fresh, was) : fresh;
  const int k = exponent_of(scale);
#pragma unroll
  for (int m = 0; m < NCH; ++m) {
    const int i = threadIdx.x + m * step;
    if (i < chunks) reinterpret_cast<uint4*>(codes + static_cast<size_t>(begin) * d)[i] = encode16(x[m], pow2(-k), infinite);
  }
  if (older && scale != was) {
    uint4* old = reinterpret_cast<uint4*>(codes + static_cast<size_t>(b) * c.B * d);
    const int j = exponent_of(was) - k;
    for (int i = threadIdx.x; i < (begin - b * c.B) * per; i += step) old[i] = rescale16(old[i], j);
  }
  if (threadIdx.x == 0) scales[b] = scale;
  if (!of_v && c.w)
    for (int t = begin + threadIdx.x; t < end; t += step) c.w[row * c.cap + t] = 0.0f;
}

// ---- eviction ----
// Weights as unsigned numbers of the same order, NaN the least, zeros of both signs the same.
__device__ __forceinline__ unsigned order_key(float w) {
  if (w != w) return 0u;
  const unsigned u = w == 0.0f ? 0u : __float_as_uint(w);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
constexpr int kSelThreads = 1024, kBins = 2048;
constexpr int kMove = 128;      // tokens that a CTA of the move takes, a multiple of every block
constexpr int kMoveThreads = 256;

struct EvictScratch {
  unsigned* ticket;  // pieces handed out so far
  unsigned* loaded;  // [pieces of a head][entries][kv heads][keys, values]: the piece's tokens are in registers
};

// The kept tokens of one (entry, head), in order.  The smallest kept weight is found by digits, 11, 11 and 10 bits from the top: a histogram of
// the next digit of the keys that agree with the digits found so far.  Each warp has a stretch of the candidates, in registers up to 32 PER of them (of
// more they are read again for every digit).  A chain of short steps: 700 candidates 5.6 us, 16 x 8 heads of up to 7680 14 us.
template <int PER>
__global__ void __launch_bounds__(kSelThreads) cache8_select_kernel(const Cache8 c, int keep, int recent, int* kept, const EvictScratch x, const SeqDesc* seqs) {
  __shared__ int hist[kBins], sums[32], found[2], warp_gt[32], warp_eq[32];
  const int head = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  pdl_wait();
  const SeqDesc sq = seqs[blockIdx.y];
  const int pieces = (keep + kMove - 1) / kMove;
  for (int i = tid; i < 2 * pieces; i += kSelThreads)
    x.loaded[(static_cast<size_t>(i >> 1) * gridDim.y + blockIdx.y) * 2 * c.H + 2 * head + (i & 1)] = 0;
  if (blockIdx.x == 0 && blockIdx.y == 0 && tid == 0) *x.ticket = 0;
  int* out = kept + (static_cast<size_t>(blockIdx.y) * c.H + head) * keep;
  const bool ok = sq.slot >= 0 && sq.slot < c.slots && sq.pos >= 0 && sq.pos <= c.cap;
  const int len = ok ? sq.pos : 0;
  if (len <= keep) {
    for (int i = tid; i < keep; i += kSelThreads) out[i] = i < len ? i : -1;
    return;
  }
  const float* w = c.w + (static_cast<size_t>(sq.slot) * c.H + head) * c.cap;
  const int cand = len - recent, want = keep - recent;
  const int stretch = (cand + 1023) / 1024 * 32, first = min(cand, warp * stretch), last = min(cand, first + stretch);
  const bool held = stretch <= 32 * PER;
  unsigned own[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) own[i] = first + 32 * i + lane < last ? order_key(w[first + 32 * i + lane]) : 0u;
  // f(key, place, there) for this lane's candidates; every lane of the warp is there each time
  auto each = [&](auto&& f) {
    if (held) {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (first + 32 * i < last) f(own[i], first + 32 * i + lane, first + 32 * i + lane < last);
    } else {
#pragma unroll 4
      for (int i = first; i < last; i += 32) f(i + lane < last ? order_key(w[i + lane]) : 0u, i + lane, i + lane < last);
    }
  };
  unsigned prefix = 0;
  int left = want;  // of the keys that agree with the prefix, the `left` largest are kept
  if (want > 0) {
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      hist[tid] = hist[tid + 1024] = 0;
      __syncthreads();
      each([&](unsigned key, int, bool there) {
        if (there && (pass == 0 || key >> (shift + bits) == prefix)) atomicAdd(&hist[(key >> shift) & ((1u << bits) - 1)], 1);
      });
      __syncthreads();
      // counts from the largest digit down: thread t has digits 2047 - 2t and 2046 - 2t
      const int hi = hist[kBins - 1 - 2 * tid], lo = hist[kBins - 2 - 2 * tid];
      int run = hi + lo;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += up;
      }
      if (lane == 31) sums[warp] = run;
      __syncthreads();
      const int before = __reduce_add_sync(0xffffffffu, lane < warp ? sums[lane] : 0), above = run - hi - lo + before;
      if (above < left && left <= above + hi) { found[0] = kBins - 1 - 2 * tid; found[1] = above; }
      else if (above + hi < left && left <= above + hi + lo) { found[0] = kBins - 2 - 2 * tid; found[1] = above + hi; }
      __syncthreads();
      prefix = prefix << bits | static_cast<unsigned>(found[0]);
      left -= found[1];
    }
  }
  // count, then write behind what the warps before keep
  int gt = 0, eq = 0;
  each([&](unsigned key, int, bool there) {
    gt += __popc(__ballot_sync(0xffffffffu, there && want > 0 && key > prefix));
    eq += __popc(__ballot_sync(0xffffffffu, there && want > 0 && key == prefix));
  });
  if (lane == 0) { warp_gt[warp] = gt; warp_eq[warp] = eq; }
  __syncthreads();
  int above = __reduce_add_sync(0xffffffffu, lane < warp ? warp_gt[lane] : 0), ties = __reduce_add_sync(0xffffffffu, lane < warp ? warp_eq[lane] : 0);
  each([&](unsigned key, int place, bool there) {
    const unsigned g = __ballot_sync(0xffffffffu, there && want > 0 && key > prefix), e = __ballot_sync(0xffffffffu, there && want > 0 && key == prefix);
    const unsigned below = (1u << lane) - 1;
    const int tie = ties + __popc(e & below), at = above + __popc(g & below) + min(tie, left);
    if ((g >> lane & 1) || ((e >> lane & 1) && tie < left)) out[at] = place;
    above += __popc(g);
    ties += __popc(e);
  });
  for (int i = tid; i < recent; i += kSelThreads) out[want + i] = cand + i;
}

// Kept tokens to the front, in place and in parallel: a piece is 128 places of a head's keys or values, whose tokens come from there or from behind.
// So a piece must not be written before the pieces in front of it have been read, which may be from there.  Pieces are handed out in
// their order: a CTA reads its tokens into registers, says so, and waits, before it writes, for those in front; whoever has one of these either has
// said so or is about to, waiting at most for pieces further in front.  Each byte is read once and written once; tokens that stay where and what
// they are are not written.  A piece is a chain of dependent accesses (number, indices, tokens, flags, writes; 17000 clocks with a CTA for
// each, 88 us for 16 x 8 heads of up to 4096 kept tokens), so CTAs stay, and ask for the next piece and its indices while they work on one: 62 us, 67
// with the flags released.
__global__ void __launch_bounds__(kMoveThreads, 4) cache8_move_kernel(const Cache8 c, int keep, int n_seqs, unsigned pieces, const int* kept, const EvictScratch x,
                                                                      const SeqDesc* seqs, int* err) {
  constexpr int kMost = kMove * kCache8Head / 16 / kMoveThreads;
  __shared__ unsigned sm_top[2][kMove / 16], sm_ticket;
  __shared__ int sm_number, sm_who, sm_entry;  // the ticket's piece: thread 0 divides
  __shared__ int sm_failed;
  const int heads = 2 * c.H;
  struct Piece { int number, who, entry, head, of_v, t0, tokens; size_t row; } p{};
  int from[kMost];  // where the tokens of this thread's 16-byte pieces are
  auto width = [&]() { return p.of_v ? c.V : c.D; };
  auto token_of = [&](int i, int per) { return per == 8 ? i >> 3 : i / per; };
  auto hand_out = [&](unsigned ticket) {
    sm_ticket = ticket;
    sm_number = static_cast<int>(ticket / static_cast<unsigned>(n_seqs * heads));
    sm_who = static_cast<int>(ticket) - sm_number * n_seqs * heads;
    sm_entry = sm_who / heads;
  };
  auto take = [&]() {  // the piece that was handed out, and its indices under way
    p.number = sm_number;
    p.who = sm_who;
    const int e = p.entry = sm_entry;
    p.head = (p.who - e * heads) >> 1;
    p.of_v = p.who & 1;
    p.t0 = p.number * kMove;
    const SeqDesc sq = seqs[e];
    p.tokens = 0;
    if (sq.slot < 0 || sq.slot >= c.slots || sq.pos < 0 || sq.pos > c.cap) return;
    p.tokens = max(0, min(kMove, min(sq.pos, keep) - p.t0));  // (compared with thread numbers, which have no sign)
    p.row = static_cast<size_t>(sq.slot) * c.H + p.head;
    const int per = width() / 16, chunks = p.tokens * per;
    const int* index = kept + (static_cast<size_t>(e) * c.H + p.head) * keep + p.t0;
    if (chunks > 0)
#pragma unroll
      for (int m = 0; m < kMost; ++m) from[m] = index[token_of(min(static_cast<int>(threadIdx.x) + m * kMoveThreads, chunks - 1), per)];
  };
  pdl_wait();
  if (threadIdx.x == 0) {
    hand_out(atomicAdd(x.ticket, 1u));
    sm_failed = 0;
  }
  if (threadIdx.x < 2 * (kMove / 16)) sm_top[threadIdx.x / (kMove / 16)][threadIdx.x % (kMove / 16)] = 0u;
  __syncthreads();
  unsigned ticket = sm_ticket;
  if (ticket < pieces) take();
  for (int round = 0; ticket < pieces; ++round) {
    const Piece q = p;
    const int d = width(), per = d / 16, chunks = q.tokens * per;
    uint8_t* codes = (q.of_v ? c.v : c.k) + q.row * c.cap * d;
    float* scales = (q.of_v ? c.vs : c.ks) + q.row * c.blocks;
    float* w = c.w + q.row * c.cap;
    unsigned* top = sm_top[round & 1];
    uint4 v[kMost];
    int ks[kMost];  // exponents of the tokens' scales; where they stay, kStays more
    constexpr int kStays = 1024;
    float wt = 0.0f;
    // (a thread without a 16-byte piece of its own reads the last one again: straight-line code, all loads at once)
    if (q.tokens > 0) {
      float sc[kMost];
#pragma unroll
      for (int m = 0; m < kMost; ++m) {
        const int i = min(static_cast<int>(threadIdx.x) + m * kMoveThreads, chunks - 1), t = token_of(i, per);
        v[m] = *reinterpret_cast<const uint4*>(codes + static_cast<size_t>(from[m]) * d + (i - t * per) * 16);
        sc[m] = scales[from[m] >> c.shift];
      }
#pragma unroll
      for (int m = 0; m < kMost; ++m) {
        const int i = min(static_cast<int>(threadIdx.x) + m * kMoveThreads, chunks - 1);
        ks[m] = exponent_of(sc[m]) + (from[m] == q.t0 + token_of(i, per) ? kStays : 0);
      }
    }
    if (!q.of_v && static_cast<int>(threadIdx.x) < q.tokens) wt = w[kept[(static_cast<size_t>(q.entry) * c.H + q.head) * keep + q.t0 + threadIdx.x]];
    unsigned next = 0;
    if (threadIdx.x == 0) next = atomicAdd(x.ticket, 1u);
#pragma unroll
    for (int m = 0; m < kMost; ++m) {
      if (q.tokens == 0) break;
      const int i = min(static_cast<int>(threadIdx.x) + m * kMoveThreads, chunks - 1), block = token_of(i, per) >> c.shift;
      const unsigned bits = __float_as_uint(top_of(v[m]) * pow2(ks[m] > 512 ? ks[m] - kStays : ks[m]));  // (>= 0: ordered like its bits)
      if (per == 8) {  // a warp's four tokens lie in one block
        const unsigned most = __reduce_max_sync(0xffffffffu, bits);
        if ((threadIdx.x & 31) == 0) atomicMax(&top[block], most);
      } else {
        atomicMax(&top[block], bits);
      }
    }
    if (threadIdx.x == 0) hand_out(next);
    asm volatile("" ::"f"(wt) : "memory");
    __syncthreads();  // every load of the CTA has arrived: what they gave has been used
    unsigned* flags = x.loaded + q.who;
    const size_t stride = static_cast<size_t>(n_seqs) * heads;
    // Released, so that the reads come before whatever the one who sees the flag writes: 5 us of 80 for 16 x 8 heads of 4096 kept tokens, as it waits for the
    // last piece's stores too.
    if (threadIdx.x == 0 && q.tokens > 0) asm volatile("st.release.gpu.global.u32 [%0], 1;" ::"l"(flags + q.number * stride) : "memory");
    ticket = sm_ticket;
    if (ticket < pieces) take();
    if (threadIdx.x < 32 && q.tokens > 0) {
      bool fine = true;
      uint64_t since = 0;
      for (int f = threadIdx.x; f < q.number && fine; f += 32)
        for (unsigned it = 0;; ++it) {
          unsigned there;
          asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(there) : "l"(flags + f * stride) : "memory");
          if (there) break;
          if ((it & 63) == 63) {
            const uint64_t now = global_timer_ns();
            if (since == 0) since = now;
            if (*reinterpret_cast<volatile int*>(err) != 0 || now - since > kWaitLimitNs) {
              atomicCAS(err, 0, DEVERR_CACHE_MOVE);
              fine = false;
              break;
            }
          }
        }
      if (!fine) sm_failed = 1;
    }
    __syncthreads();
    if (sm_failed) return;
#pragma unroll
    for (int m = 0; m < kMost; ++m) {
      const int i = threadIdx.x + m * kMoveThreads;
      if (i >= chunks) continue;
      const int k = scale_exponent(__uint_as_float(top[token_of(i, per) >> c.shift]));
      if (ks[m] == k + kStays) continue;
      reinterpret_cast<uint4*>(codes + static_cast<size_t>(q.t0) * d)[i] = rescale16(v[m], (ks[m] > 512 ? ks[m] - kStays : ks[m]) - k);
    }
    if (static_cast<int>(threadIdx.x) < (q.tokens + c.B - 1) >> c.shift) scales[(q.t0 >> c.shift) + threadIdx.x] = pow2(scale_exponent(__uint_as_float(top[threadIdx.x])));
    if (!q.of_v && static_cast<int>(threadIdx.x) < q.tokens) w[q.t0 + threadIdx.x] = wt;
    // the other round's maxima: everyone has passed two barriers since they were read
    if (threadIdx.x < kMove / 16) sm_top[(round & 1) ^ 1][threadIdx.x] = 0u;
    __syncthreads();
  }
}

}  // namespace

int cache8_append(const Cache8& c, const Cache8Append& a, const SeqDesc* seqs, int n_seqs, int max_len, cudaStream_t st) {
  const int size = a.f32 ? 4 : 2;
  const uintptr_t rows16 = reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) | static_cast<uintptr_t>(a.ldk * size) |
                           static_cast<uintptr_t>(a.ldv * size);
  const int vec = (rows16 & 15) == 0;
  const dim3 grid((max_len + c.B - 2) / c.B + 1, 2 * c.H, n_seqs);
  // pieces of a block, and as many threads as leave each a few of them
  const int most = (max_len < c.B ? max_len : c.B) * ((c.D > c.V ? c.D : c.V) / 16);
  auto go = [&](auto kernel, int threads) { launch_kernel(kernel, grid, dim3(threads), 0, st, 1, c, a, seqs, max_len, vec); };
  if (most <= 64) a.f32 ? go(cache8_append_kernel<float, 1>, 64) : go(cache8_append_kernel<bf16, 1>, 64);
  else if (most <= 512) a.f32 ? go(cache8_append_kernel<float, 2>, 256) : go(cache8_append_kernel<bf16, 2>, 256);
  else a.f32 ? go(cache8_append_kernel<float, 4>, 256) : go(cache8_append_kernel<bf16, 4>, 256);
  return static_cast<int>(cudaGetLastError());
}

size_t cache8_evict_scratch_bytes(const Cache8& c, int n_seqs, int keep) {
  return TEENY_CACHE8_COUNTER_BYTES + 256 + static_cast<size_t>((keep + kMove - 1) / kMove) * n_seqs * 2 * c.H * 4;
}

int cache8_evict(const Cache8& c, int keep, int recent, int* kept, void* scratch, const SeqDesc* seqs, const SeqDesc* host, int n_seqs, cudaStream_t st) {
  int* err = device_error_word();
  if (!err) return TEENY_ERR_DRIVER;
  const long long pieces = static_cast<long long>((keep + kMove - 1) / kMove) * n_seqs * 2 * c.H;
  if (pieces > 0x7fffffffLL) return TEENY_ERR_BAD_ARG;
  // (the place of the attention's counters is left alone: the calls may share scratch)
  uint8_t* own = static_cast<uint8_t*>(scratch) + TEENY_CACHE8_COUNTER_BYTES;
  const EvictScratch x{reinterpret_cast<unsigned*>(own), reinterpret_cast<unsigned*>(own + 256)};
  auto select = [&](auto kernel) { launch_kernel(kernel, dim3(c.H, n_seqs), dim3(kSelThreads), 0, st, 1, c, keep, recent, kept, x, seqs); };
  int most = 0;  // candidates
  for (int i = 0; host && i < n_seqs; ++i) most = host[i].pos - recent > most ? host[i].pos - recent : most;
  if (host && most <= 2 * kSelThreads) select(cache8_select_kernel<2>);
  else select(cache8_select_kernel<16>);
  const bool pdl = pdl_enabled();
  pdl_set_enabled(true);
  const long long stay = 4ll * sm_count();
  launch_kernel(cache8_move_kernel, dim3(static_cast<unsigned>(pieces < stay ? pieces : stay)), dim3(kMoveThreads), 0, st, 1, c, keep, n_seqs,
                static_cast<unsigned>(pieces), static_cast<const int*>(kept), x, seqs, err);
  pdl_set_enabled(pdl);
  return static_cast<int>(cudaGetLastError());
}

namespace {

bool cache_of(const teeny_cache8_shape* s, Cache8* c) {
  if (!s || s->slots <= 0 || s->kv_heads <= 0 || s->kv_heads > 16384 || s->max_cached <= 0 || s->max_cached > (1 << 30) || s->dim <= 0 ||
      s->dim > kCache8Head || s->dim % 16 || s->vdim <= 0 || s->vdim > kCache8Head || s->vdim % 16 ||
      (s->block != 16 && s->block != 32 && s->block != 64 && s->block != 128))
    return false;
  *c = Cache8{nullptr, nullptr, nullptr, nullptr, nullptr, s->slots, s->kv_heads, s->max_cached, s->dim, s->vdim, s->block,
              (s->max_cached + s->block - 1) / s->block,
              s->block == 16 ? 4 : s->block == 32 ? 5 : s->block == 64 ? 6 : 7};
  return true;
}
int bind_cache(Cache8* c, void* k, void* v, float* ks, float* vs, float* w) {
  if (!k || !v || !ks || !vs) return TEENY_ERR_BAD_ARG;
  if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) return TEENY_ERR_ALIGNMENT;
  c->k = static_cast<uint8_t*>(k);
  c->v = static_cast<uint8_t*>(v);
  c->ks = ks;
  c->vs = vs;
  c->w = w;
  return TEENY_OK;
}
// The host's copy of a step table, where the caller has one.  once: a slot may come only once (with by_len: in entries that have tokens).
int check_table(const SeqDesc* t, int n, const Cache8& c, bool once, bool by_len) {
  unsigned char* seen = once && n > 1 ? static_cast<unsigned char*>(calloc((static_cast<size_t>(c.slots) + 7) / 8, 1)) : nullptr;
  if (once && n > 1 && !seen) return TEENY_ERR_BAD_ARG;
  int rc = TEENY_OK;
  for (int i = 0; i < n && rc == TEENY_OK; ++i) {
    if (t[i].slot < 0 || t[i].slot >= c.slots) { rc = TEENY_ERR_BAD_ARG; break; }
    if (!seen || (by_len && t[i].len == 0)) continue;
    unsigned char& byte = seen[t[i].slot >> 3];
    const unsigned char bit = static_cast<unsigned char>(1u << (t[i].slot & 7));
    if (byte & bit) rc = TEENY_ERR_BAD_ARG;
    byte |= bit;
  }
  free(seen);
  return rc;
}
// (an entry without tokens does nothing)
bool all_fit(const SeqDesc* t, int n, const Cache8& c, int rows, int max_len) {
  for (int i = 0; i < n; ++i)
    if (!cache8_fits(t[i], c, rows, max_len) && !(t[i].len == 0 && t[i].pos >= 0 && t[i].pos <= c.cap)) return false;
  return true;
}
// No row is two entries' (both would write its results).
bool rows_apart(const SeqDesc* t, int n, int rows) {
  int end = 0, i = 0;
  for (; i < n && (t[i].len == 0 || t[i].row0 >= end); ++i)
    if (t[i].len > 0) end = t[i].row0 + t[i].len;
  if (i == n) return true;
  // (not in order)
  unsigned char* seen = static_cast<unsigned char*>(calloc(rows, 1));
  bool apart = seen != nullptr;
  for (i = 0; i < n && apart; ++i)
    for (int r = t[i].row0; r < t[i].row0 + t[i].len && apart; ++r) {
      apart = !seen[r];
      seen[r] = 1;
    }
  free(seen);
  return apart;
}
// The longest entry that can fit, where the caller's bound is above it.
int longest_of(int max_len, const Cache8& c, int rows) { return std::min(max_len, std::min(c.cap, rows)); }
bool step_sizes(int rows, int n_seqs, int max_len) { return rows > 0 && n_seqs > 0 && n_seqs <= 65535 && max_len > 0; }

}  // namespace
}  // namespace teeny

using namespace teeny;

extern "C" {

int teeny_cache8_append(int f32, const teeny_cache8_shape* shape, void* k, void* v, float* k_scale, float* v_scale, float* weights,
                        const void* k_new, long long ldk, const void* v_new, long long ldv, int rows, const int* seqs,
                        const int* host_seqs, int n_seqs, int max_len, teeny_stream_t stream) {
  Cache8 c;
  if (!cache_of(shape, &c) || !k_new || !v_new || !seqs || !step_sizes(rows, n_seqs, max_len) ||
      ldk < static_cast<long long>(c.H) * c.D || ldv < static_cast<long long>(c.H) * c.V)
    return TEENY_ERR_BAD_ARG;
  if (const int rc = bind_cache(&c, k, v, k_scale, v_scale, weights)) return rc;
  if (const SeqDesc* host = reinterpret_cast<const SeqDesc*>(host_seqs)) {
    if (!all_fit(host, n_seqs, c, rows, max_len)) return TEENY_ERR_BAD_ARG;
    if (const int rc = check_table(host, n_seqs, c, true, true)) return rc;
  }
  const Cache8Append a{f32 != 0, k_new, v_new, ldk, ldv, rows};
  return cache8_append(c, a, reinterpret_cast<const SeqDesc*>(seqs), n_seqs, longest_of(max_len, c, rows), reinterpret_cast<cudaStream_t>(stream));
}

size_t teeny_cache8_attention_scratch_bytes(const teeny_cache8_shape* shape, int f32, int heads, int rows, int n_seqs, int max_len,
                                            int with_weights) {
  Cache8 c;
  if (!cache_of(shape, &c) || heads <= 0 || heads % c.H || !step_sizes(rows, n_seqs, max_len)) return 0;
  return cache8_attention_scratch_bytes(c, f32 != 0, heads, rows, n_seqs, longest_of(max_len, c, rows), with_weights != 0);
}

int teeny_cache8_attention(int f32, const teeny_cache8_shape* shape, const void* k, const void* v, const float* k_scale,
                           const float* v_scale, float* weights, float weight_decay, const void* q, long long ldq, void* out,
                           long long ldo, int rows, int heads, float score_scale, float softcap, const float* sink, const void* gate,
                           long long ldg, float* lse, void* scratch, size_t scratch_bytes, const int* seqs, const int* host_seqs,
                           int n_seqs, int max_len, teeny_stream_t stream) {
  Cache8 c;
  if (!cache_of(shape, &c) || !q || !out || !seqs || !step_sizes(rows, n_seqs, max_len) || heads <= 0 || heads % c.H ||
      ldq < static_cast<long long>(heads) * c.D || ldo < static_cast<long long>(heads) * c.V ||
      (gate && ldg < static_cast<long long>(heads) * c.V) || !(softcap == 0.0f || (softcap > 1e-30f && softcap < 1e30f)) || !(score_scale > -1e30f && score_scale < 1e30f))
    return TEENY_ERR_BAD_ARG;
  if (const int rc = bind_cache(&c, const_cast<void*>(k), const_cast<void*>(v), const_cast<float*>(k_scale), const_cast<float*>(v_scale), weights))
    return rc;
  if (const SeqDesc* host = reinterpret_cast<const SeqDesc*>(host_seqs)) {
    if (!all_fit(host, n_seqs, c, rows, max_len) || !rows_apart(host, n_seqs, rows)) return TEENY_ERR_BAD_ARG;
    if (const int rc = check_table(host, n_seqs, c, weights != nullptr, true)) return rc;
  }
  max_len = longest_of(max_len, c, rows);
  const size_t need = cache8_attention_scratch_bytes(c, f32 != 0, heads, rows, n_seqs, max_len, weights != nullptr);
  if (need && (!scratch || scratch_bytes < need)) return TEENY_ERR_SCRATCH;
  if (reinterpret_cast<uintptr_t>(scratch) & 31) return TEENY_ERR_ALIGNMENT;  // (prompts' tokens are widened by stores of 32 bytes)
  const Cache8Attn a{f32 != 0, q, ldq, out, ldo, rows, heads, score_scale, softcap, sink, gate, ldg, lse, weights != nullptr, weight_decay,
                     scratch};
  return cache8_attention(c, a, reinterpret_cast<const SeqDesc*>(seqs), n_seqs, max_len, reinterpret_cast<cudaStream_t>(stream));
}

size_t teeny_cache8_evict_scratch_bytes(const teeny_cache8_shape* shape, int n_seqs, int keep) {
  Cache8 c;
  if (!cache_of(shape, &c) || n_seqs <= 0 || n_seqs > 65535 || keep <= 0 || keep > c.cap) return 0;
  return cache8_evict_scratch_bytes(c, n_seqs, keep);
}

int teeny_cache8_evict(const teeny_cache8_shape* shape, void* k, void* v, float* k_scale, float* v_scale, float* weights, int keep,
                       int recent, int* kept, void* scratch, size_t scratch_bytes, const int* seqs, const int* host_seqs, int n_seqs,
                       teeny_stream_t stream) {
  Cache8 c;
  if (!cache_of(shape, &c) || !weights || !kept || !seqs || n_seqs <= 0 || n_seqs > 65535 || keep <= 0 || keep > c.cap || recent < 0 || recent > keep)
    return TEENY_ERR_BAD_ARG;
  if (const int rc = bind_cache(&c, k, v, k_scale, v_scale, weights)) return rc;
  if (const SeqDesc* host = reinterpret_cast<const SeqDesc*>(host_seqs)) {
    for (int i = 0; i < n_seqs; ++i)
      if (host[i].pos < 0 || host[i].pos > c.cap) return TEENY_ERR_BAD_ARG;
    if (const int rc = check_table(host, n_seqs, c, true, false)) return rc;
  }
  const size_t need = cache8_evict_scratch_bytes(c, n_seqs, keep);
  if (need && (!scratch || scratch_bytes < need)) return TEENY_ERR_SCRATCH;
  if (reinterpret_cast<uintptr_t>(scratch) & 15) return TEENY_ERR_ALIGNMENT;
  return cache8_evict(c, keep, recent, kept, scratch, reinterpret_cast<const SeqDesc*>(seqs), reinterpret_cast<const SeqDesc*>(host_seqs), n_seqs,
                      reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
