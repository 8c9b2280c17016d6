// Causal attention over the 8-bit key/value cache (layout in teeny_cache8.h) for any number of query rows, and the weights that the cached tokens
// receive.
//
// Both products run on f16 operands with f32 sums (mma.sync m16n8k16): an E4M3 number is an f16 number exactly, and one conversion makes two of
// them.  (mma.sync on E4M3 operands is made of the same f16 products here, with additions of its own behind each: 0.19 m16n8k32 a clock
// and SM, where the f16 pairs run at 0.42 / 2.)  The 16 rows of a product are keys, then dimensions of the values; its eight columns are query rows,
// so that few query heads waste nothing.  A query row is scaled by a power of two so that its largest number is in [2^14, 2^15): a bf16
// number below 2^-28 of that loses bits, no other.  f32 rows are two f16 terms, 22 bits, in two column tiles whose sums lie in the same thread's
// registers.  Probabilities are f16 numbers times 2^14 (f32: two terms as well), so that a key is lost only 2^-38 below the row's
// maximum so far.  Scales of key blocks multiply the scores; those of value blocks, relative to the largest so far (2^-112 at least), the probabilities.
//
// The call is bound by reading the cache.  A CTA is four warps, each with slices of 32 keys of its own in flight (keys and values by TMA, their scales by
// 4-byte asynchronous copies on the same barrier).  Work is divided evenly by slices: entry after entry, head after head, row group after row
// group, each CTA takes the same number of consecutive slices of all of them, whatever the lengths, and its warps take them in turn.  Where
// a sequence ends or a share does, the warps' sums are added through shared memory.  A sequence that lies in several CTAs' shares leaves partial
// results in scratch, at most two for each CTA; the last one to have stored its part adds them (a second kernel for it cost 4 to 10 us a
// call; parts of single warps, four times as many, up to 14 us).  No CTA waits for another.  64 sequences of 1500 to 6000 tokens, 32 / 8 heads of 128, 500 MB:
// 92 us, 5.4 TB/s; one of 701 tokens: 10.0 us, a chain of latencies.
#include <atomic>
#include <type_traits>

#include "../../include/teeny_cache8.h"
#include "common.cuh"
#include "kernels.h"
#include "mma.cuh"

namespace teeny {

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr int kSlice = 32;                     // keys that a warp takes at a time
constexpr int kBox = kSlice * kCache8Head;     // 4 KB: their keys, or their values (narrower heads are filled up with zeros by the copies)
constexpr int kStage = 2 * kBox;
constexpr int kWarps = 4;                      // of a CTA
// The values' reference begins here: a block of zeros has the scale 2^-126, and 2^14 over that is no f32 number, while 2^14 / kLeastRef and kLeastRef / 2^14 are
// normal ones.  Blocks of smaller scales (numbers below 2^-103) lose bits where a probability is below 2^-14.
constexpr float kLeastRef = 0x1p-112f;

// Variant of the kernel: RT tiles of eight query rows in TERMS f16 terms (bf16: 1, f32: 2).  One tile in one term fits 168 registers, with which an SM
// has three CTAs; more take two.
template <int RT_, int TERMS_>
struct Variant {
  static constexpr int RT = RT_, TERMS = TERMS_, NT = RT * TERMS, kRows = 8 * RT, kCtas = NT == 1 ? 3 : 2, kStages = 2;
  using T = typename std::conditional<TERMS == 2, float, bf16>::type;
  // shared memory: stages of the warps, scales f32 [warps][stages][4], int [128] first NaN value of each dimension, maximum and sum of a row [2][warps][rows][2],
  // barriers, factors [rows], queries uint2 [row tiles][8 steps][32 lanes] (one row tile: in registers), sums on their way f32 [2][RT * 32][32 lanes]
  static constexpr int kScales = kWarps * kStages * kStage;
  static constexpr int kNan = kScales + kWarps * kStages * 16;
  static constexpr int kML = kNan + 128 * 4;
  static constexpr int kBars = kML + 2 * kWarps * kRows * 8;
  static constexpr int kFactor = kBars + kWarps * kStages * 8;
  static constexpr int kQ = kFactor + kRows * 4;
  static constexpr int kMerge = kQ + (RT == 1 ? 0 : RT * 8 * 32 * 8);
  static constexpr int kBytes = kMerge + 2 * RT * 32 * 32 * 4 + 1024;
  static_assert((kBytes + 1024) * kCtas <= 233472, "shared memory");
};

// D (16 x 8) += A (16 x 16) B
__device__ __forceinline__ void mma_f16_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8 x 8 16-bit numbers: lane (g, c) gives (row g, columns 2c, 2c + 1) and gets (rows 2c, 2c + 1 of column g)
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// Four E4M3 numbers as two f16 pairs
__device__ __forceinline__ void widen(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// what the f16 numbers `two` leave of x and y, times 2^11
__device__ __forceinline__ uint32_t rest_f16x2(uint32_t two, float x, float y) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&two));
  return pack_f16x2((x - f.x) * 2048.0f, (y - f.y) * 2048.0f);
}
__device__ __forceinline__ float load_one(const bf16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load_one(const float* p) { return *p; }
__device__ __forceinline__ void store_one(bf16* p, float x) { *p = __float2bfloat16_rn(x); }
__device__ __forceinline__ void store_one(float* p, float x) { *p = x; }

struct Shared {  // what a call's kernels share
  Cache8 c;
  Cache8Attn a;
  const SeqDesc* seqs;
  int n_seqs, max_len, G;
  float scale_log2, one_over_cap, cap_l2;  // (the cap in base 2, like the scores)
  float* part_o;   // [2 * CTAs][rows of a unit][128]
  float* part_ml;  // [2 * CTAs][rows of a unit][2]
  unsigned* arrivals;  // [CTAs]: how many have stored their part of the unit that begins in a CTA's share and goes on behind it, zero between calls
  float* lse2;     // [rows][Hq], base 2, or null
  float* scores;   // [entries][Hq][score_row] base 2, or null
  int score_row;   // cap, rounded up to whole fours
  int parts;       // CTAs of the main kernel
  int vec_q, vec_o;
  int* err;
};

// Slices of an entry: its units are (head, row group), each over all its slices.  (All counts of a call fit 31 bits, the host sees to that: divisions
// of 64-bit numbers, a hundred instructions each, made up most of a short call.)
struct EntryShape { int slices, groups, all; };
__device__ __forceinline__ EntryShape entry_shape(const Shared& s, const SeqDesc& sq, int rows) {
  EntryShape e{0, 0, 0};
  if (!cache8_fits(sq, s.c, s.a.rows, s.max_len)) return e;
  e.slices = (sq.pos + sq.len + kSlice - 1) / kSlice;
  e.groups = (sq.len * s.G + rows - 1) / rows;
  e.all = e.slices * e.groups * s.c.H;
  return e;
}
// How the slices are shared.  With many units each of the CTAs takes the same number of consecutive slices, whatever units they are of: the first `more`
// take one more than the others' `each`.  With few units, a unit is cut into parts of `cut` slices and each CTA takes one: the end
// of a unit inside a share costs a CTA 5000 clocks (eight kv heads, one sequence of 701 tokens: 12.9 us without, 9.8 with; four of 14050: 27.1 and 21.8; four of
// 40001 with weights: 82.3 and 80.3; 16 x 5 tokens, ragged: 41.8 and 38.2, by now 39.0).  No share is less than a slice for each warp (unless its unit is), nor are there many more than 64 to a
// unit, whose parts have to be added again.
struct Shares {
  int parts, each, more, cut;
  __device__ __forceinline__ Shares(int most, int total, int units) {
    const int least = max(kWarps, total / 64 / units);
    cut = units * 2 <= most ? max(least, (total + most - units - 1) / (most - units)) : 0;
    parts = min(most, max((total + least - 1) / least, min(units, total)));
    each = total / parts;
    more = total - parts * each;
  }
  __device__ __forceinline__ int begin(int part) const { return part * each + min(part, more); }
  __device__ __forceinline__ int owner(int slice) const {
    const int big = more * (each + 1);
    return slice < big ? slice / (each + 1) : more + (slice - big) / each;
  }
  __device__ __forceinline__ int cuts(int slices) const { return (slices + cut - 1) / cut; }
};

__device__ __forceinline__ int warp_sum_int(int v) { return static_cast<int>(__reduce_add_sync(0xffffffffu, static_cast<unsigned>(v))); }

__device__ __forceinline__ void note_lse(const Shared& s, size_t row, int h, float lse2) {
  if (s.lse2) s.lse2[row * s.a.Hq + h] = lse2;
  if (s.a.lse) s.a.lse[row * s.a.Hq + h] = lse2 * kLn2;
}
// The results of row r (counted in its entry) of kv head hk, dimensions 4 lane ..: x unnormalised, relative to the maximum m (base 2), l the row sum.
template <typename T>
__device__ __forceinline__ void finish_row(const Shared& s, const SeqDesc& sq, int hk, int r, int lane, const float4& x, float m, float l) {
  const int i = r / s.G, hq = hk * s.G + r - i * s.G;
  const size_t row = static_cast<size_t>(sq.row0) + i;
  float inv = 1.0f;
  if (s.a.sink) {
    const float sink = s.a.sink[hq], over = fmaf(sink, kLog2e, -m);
    if (over > 0.0f) {  // relative to the sink: its exponential relative to the scores may be no f32 number
      inv = ex2(-over);
      l = fmaf(l, inv, 1.0f);
      m = sink * kLog2e;
    } else {
      l += ex2(over);
    }
  }
  if (lane == 0) note_lse(s, row, hq, m + log2f(l));
  if (4 * lane >= s.c.V) return;
  inv /= l;
  float y[4] = {x.x * inv, x.y * inv, x.z * inv, x.w * inv};
  if (s.a.gate) {
    const T* gate = static_cast<const T*>(s.a.gate) + row * s.a.ldg + static_cast<size_t>(hq) * s.c.V + 4 * lane;
#pragma unroll
    for (int d = 0; d < 4; ++d) y[d] *= sigmoid_f(load_one(gate + d));
  }
  T* out = static_cast<T*>(s.a.out) + row * s.a.ldo + static_cast<size_t>(hq) * s.c.V + 4 * lane;
  if (s.vec_o) {
    if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(out) = make_uint2(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]));
    else *reinterpret_cast<float4*>(out) = make_float4(y[0], y[1], y[2], y[3]);
  } else {
#pragma unroll
    for (int d = 0; d < 4; ++d) store_one(out + d, y[d]);
  }
}

// A query row, of which this lane (c = lane % 4) has the dimensions 32 c .. 32 c + 31.
template <typename T>
__device__ __forceinline__ void load_row(const T* q, int dim, bool valid, bool vec, int c, float (&x)[32]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int d0 = 32 * c + 16 * h;
    if (!valid || d0 >= dim) {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[16 * h + i] = 0.0f;
    } else if (vec && sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint4 w = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(q) + d0 + 8 * i);
        const uint32_t r[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) { x[16 * h + 8 * i + 2 * e] = bf16_lo(r[e]); x[16 * h + 8 * i + 2 * e + 1] = bf16_hi(r[e]); }
      }
    } else if (vec) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 w = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(q) + d0 + 4 * i);
        x[16 * h + 4 * i] = w.x; x[16 * h + 4 * i + 1] = w.y; x[16 * h + 4 * i + 2] = w.z; x[16 * h + 4 * i + 3] = w.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[16 * h + i] = load_one(q + d0 + i);
    }
  }
}
// ... scaled, as f16 pairs: word w is dimensions 32 c + 2 w, + 1; term[1]: the rest.  Returns the factor that takes scores back (base 2).
template <int TERMS>
__device__ __forceinline__ float split_row(const float (&x)[32], float scale_log2, uint32_t (&term)[TERMS][16]) {
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 32; ++i) amax = fmaxf(amax, fabsf(x[i]));
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
  int p = 0;
  // (from -113 on, for the largest f32 numbers; with more than 118 the factor would be subnormal, and rows below 2^-104 are left smaller instead)
  if (amax > 0.0f && amax < INFINITY) p = min(118, 14 + 127 - static_cast<int>(__float_as_uint(amax) >> 23));
  const float up = __uint_as_float(static_cast<unsigned>(127 + p) << 23), down = __uint_as_float(static_cast<unsigned>(127 - p) << 23);
#pragma unroll
  for (int w = 0; w < 16; ++w) {
    const float a = x[2 * w] * up, b = x[2 * w + 1] * up;
    term[0][w] = pack_f16x2(a, b);
    if (TERMS > 1) term[TERMS - 1][w] = rest_f16x2(term[0][w], a, b);
  }
  return down * scale_log2;
}

// One (entry, head, row group) as far as it lies in a warp's share.
struct Piece {
  SeqDesc sq;
  int e, slices, groups, hk, rg, j, end, limit;  // slices j .. end - 1; limit: keys that the group's last row sees
  bool whole, first;
};
__device__ __forceinline__ void piece_range(const Shared& s, Piece& p, int rows, int j0, int left) {
  p.j = j0;
  p.end = min(p.slices, j0 + left);
  p.whole = j0 == 0 && p.end == p.slices;
  p.limit = p.sq.pos + (min(p.sq.len * s.G, (p.rg + 1) * rows) - 1) / s.G + 1;
}
// to the next unit, of which `left` slices may be taken
__device__ __forceinline__ void next_piece(const Shared& s, Piece& p, int rows, int left) {
  if (++p.rg == p.groups) {
    p.rg = 0;
    if (++p.hk == s.c.H) {
      p.hk = 0;
      EntryShape es;
      do {
        p.sq = s.seqs[++p.e];
        es = entry_shape(s, p.sq, rows);
      } while (es.all == 0);
      p.slices = es.slices;
      p.groups = es.groups;
    }
  }
  p.first = false;
  piece_range(s, p, rows, 0, left);
}

template <typename V>
__global__ void __launch_bounds__(32 * kWarps, V::kCtas)
cache8_attention_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v, const __grid_constant__ Shared s) {
  using T = typename V::T;
  constexpr int R = V::kRows, ST = V::kStages, RT = V::RT, TERMS = V::TERMS, NT = V::NT;
  extern __shared__ uint8_t smem_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  const uint32_t ring = base + warp * (ST * kStage), bars = base + V::kBars + warp * (ST * 8), scale_at = base + V::kScales + warp * (ST * 16);
  // units of which this CTA has left a part: its first and its last
  __shared__ struct Left { int c0, c1, slot0, e, hk, rg; } sm_left[2];  // c0 .. c1: the CTAs that have parts of it (none: c1 < c0)
  if (lane == 0) {
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
    for (int st = 0; st < ST; ++st) mbar_init(bars + 8 * st, 1 + 4);
    mbar_fence_init();
  }
  if (threadIdx.x < 2) sm_left[threadIdx.x] = Left{0, -1, 0, 0, 0, 0};
  __syncwarp();
  pdl_wait();
  // ---- this CTA's share (each warp works it out) ----
  const int part = blockIdx.x;
  int total = 0, units = 0, mine = 0;  // mine: of this lane's entry among the first 32
  for (int e = lane; e < s.n_seqs; e += 32) {
    const EntryShape es = entry_shape(s, s.seqs[e], R);
    if (e < 32) mine = es.all;
    total += es.all;
    units += es.groups * s.c.H;
  }
  total = warp_sum_int(total);
  units = warp_sum_int(units);
  if (total == 0) return;
  const Shares shares(s.parts, total, units);
  // (counted in slices, or with cut units in their parts)
  const int t0 = shares.cut ? part : part < shares.parts ? shares.begin(part) : total;
  int share, cuts = 1;
  Piece p;
  {
    int before = 0, at = 0, found = -1;
    for (int e0 = 0; found < 0; e0 += 32) {
      if (e0 >= s.n_seqs) return;  // nothing is left for this CTA
      if (e0 > 0) mine = e0 + lane < s.n_seqs ? entry_shape(s, s.seqs[e0 + lane], R).all : 0;
      if (shares.cut && mine > 0) {
        const EntryShape es = entry_shape(s, s.seqs[e0 + lane], R);
        mine = shares.cuts(es.slices) * es.groups * s.c.H;
      }
      int run = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, run, o);
        if (lane >= o) run += up;
      }
      const int end = before + run;
      const unsigned who = __ballot_sync(0xffffffffu, mine > 0 && t0 >= end - mine && t0 < end);
      before = __shfl_sync(0xffffffffu, end, 31);
      if (!who) continue;
      const int src = __ffs(who) - 1;
      found = e0 + src;
      at = t0 - __shfl_sync(0xffffffffu, end - mine, src);
    }
    p.e = found;
    p.sq = s.seqs[found];
    const EntryShape es = entry_shape(s, p.sq, R);
    p.slices = es.slices;
    p.groups = es.groups;
    if (shares.cut) cuts = shares.cuts(es.slices);
    const int per_unit = shares.cut ? cuts : es.slices, unit = at / per_unit, inside = at - unit * per_unit;
    p.hk = unit / es.groups;
    p.rg = unit - p.hk * es.groups;
    p.first = true;
    share = shares.cut ? min(shares.cut, es.slices - inside * shares.cut) : shares.begin(part + 1) - t0;
    piece_range(s, p, R, shares.cut ? inside * shares.cut : inside, share);
  }
  pdl_trigger();
  // Row g of the row tile that this warp makes ready (with one, every warp does): the first piece's is asked for in front of the cache's slices, behind
  // which it would queue for 5000 clocks.
  const int rt_mine = RT == 1 ? 0 : warp;
  float raw[32];
  auto ask_row = [&](const Piece& of) {
    if (RT > 1 && warp >= RT) return;
    const int r = of.rg * R + rt_mine * 8 + g, i = r / s.G, hq = of.hk * s.G + r - i * s.G;
    const bool valid = i < of.sq.len;
    load_row(static_cast<const T*>(s.a.q) + static_cast<size_t>(of.sq.row0 + (valid ? i : 0)) * s.a.ldq + static_cast<size_t>(hq) * s.c.D, s.c.D, valid, s.vec_q, c, raw);
  };
  ask_row(p);
  // the slices that this warp asks for: every fourth of the share
  Piece load = p;
  int load_rest = share, load_j = p.j + warp, load_at = warp, issued = 0, count = 0;
  auto load_next = [&]() {
    if (load_at >= share) return;
    while (load_j >= load.end) {
      const int over = load_j - load.end;
      load_rest -= load.end - load.j;
      next_piece(s, load, R, load_rest);
      load_j = over;
    }
    const int st = issued & (ST - 1), key0 = load_j * kSlice;
    const uint32_t bar = bars + 8 * st;
    if (lane < 4) {  // scales of the slice's two groups of 16 keys; blocks behind the last key may hold anything: zero is written
      const int key = key0 + 16 * (lane & 1);
      const uint32_t bytes = key < load.limit ? 4 : 0;
      const float* src = (lane < 2 ? s.c.ks : s.c.vs) + (static_cast<size_t>(load.sq.slot) * s.c.H + load.hk) * s.c.blocks + (bytes ? key >> s.c.shift : 0);
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n\tcp.async.mbarrier.arrive.noinc.shared::cta.b64 [%3];"
                   ::"r"(scale_at + st * 16 + lane * 4), "l"(src), "r"(bytes), "r"(bar) : "memory");
    }
    if (lane == 0) {
      mbar_expect_tx(bar, kStage);
      tma_load_4d(ring + st * kStage, &tmap_k, bar, 0, key0, load.hk, load.sq.slot);
      tma_load_4d(ring + st * kStage + kBox, &tmap_v, bar, 0, key0, load.hk, load.sq.slot);
    }
    load_j += kWarps;
    load_at += kWarps;
    ++issued;
  };
#pragma unroll
  for (int st = 0; st < ST; ++st) load_next();

  int* sm_nan = reinterpret_cast<int*>(gen + V::kNan);
  float* sm_ml = reinterpret_cast<float*>(gen + V::kML);
  float* sm_factor = reinterpret_cast<float*>(gen + V::kFactor);
  bool ok = true;
  int flip = 0, done = 0, unit_begin = t0 - p.j;  // slices of the share in front of the piece; of the call in front of its unit
  for (;;) {
    // ---- queries as B fragments: row g of tile rt is column g ----
    float factor[RT][2];      // of the rows 2c, 2c + 1, whose scores this lane gets
    int rows_limit[RT][2];    // keys that they see
    uint2 q_regs[RT == 1 ? NT * 8 : 1];
    uint32_t term[TERMS][16];
    const float f = split_row<TERMS>(raw, s.scale_log2, term);
    if (RT > 1 || p.sq.len > 1) __syncthreads();  // the piece before is finished with what is written here
    if (p.sq.len > 1) sm_nan[threadIdx.x] = 0x7fffffff;
    if (RT == 1) {
#pragma unroll
      for (int t = 0; t < TERMS; ++t)
#pragma unroll
        for (int step = 0; step < 8; ++step) q_regs[RT == 1 ? t * 8 + step : 0] = make_uint2(term[t][2 * step], term[t][2 * step + 1]);
    } else if (warp < RT) {
#pragma unroll
      for (int step = 0; step < 8; ++step)
        reinterpret_cast<uint2*>(gen + V::kQ)[(warp * 8 + step) * 32 + lane] = make_uint2(term[0][2 * step], term[0][2 * step + 1]);
      if (c == 0) sm_factor[warp * 8 + g] = f;
    }
    if (RT > 1 || p.sq.len > 1) __syncthreads();
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const int i = (p.rg * R + rt * 8 + 2 * c + z) / s.G;
        factor[rt][z] = RT == 1 ? __shfl_sync(0xffffffffu, f, (2 * c + z) * 4) : sm_factor[rt * 8 + 2 * c + z];
        rows_limit[rt][z] = i < p.sq.len ? p.sq.pos + i + 1 : p.limit;
      }

    // acc[tile][j]: dimensions 16 g + 2j (rows 2c, 2c + 1), 16 g + 2j + 1 (the same), in units of vref * 2^-14
    float m[RT][2], l[RT][2], acc[NT][8][4];
    float vref = kLeastRef;  // largest scale of the values so far
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        m[rt][z] = -INFINITY;
        l[rt][z] = 0.0f;
      }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[nt][j][0] = acc[nt][j][1] = acc[nt][j][2] = acc[nt][j][3] = 0.0f;
    int half = 0;  // 1, 2: only the slice's first, second 16 keys count
    for (int sj = p.j + ((warp - done) & (kWarps - 1)); sj < p.end && ok;) {
      const int st = count & (ST - 1), kb = sj * kSlice;
      if (!mbar_wait(bars + 8 * st, count / ST & 1, s.err, DEVERR_ATTN_SOFTMAX)) {
        ok = false;
        break;
      }
      if (kb < p.limit) {
        const uint8_t *kt = gen + warp * (ST * kStage) + st * kStage + g * 128, *vt = gen + warp * (ST * kStage) + st * kStage + kBox;
        const float4 scales = *reinterpret_cast<const float4*>(gen + V::kScales + (warp * ST + st) * 16);
        const float ks0 = scales.x, ks1 = scales.y, vs0 = scales.z;
        float vs1 = scales.w;
        const bool masked = kb + kSlice > p.sq.pos + 1;
        // Two blocks of 16, the later one of much larger values, which not all rows see: one block at a time, so that it takes no bits from the rows before it.
        // (16 entries of five tokens: 39.2 us without, 39.9 with the loop's way back; a reference for each row 43.2.)
        if (masked && p.sq.len > 1 && half == 0 && vs1 > 16.0f * vs0) half = 1;
        if (half == 1) vs1 = 0.0f;
        // ---- scores: keys 16 u + g and 16 u + 8 + g of the slice are rows g and g + 8 of tile u; lane c reads the dimensions that it holds of the query ----
        float x[NT][2][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int u = 0; u < 2; ++u) x[nt][u][0] = x[nt][u][1] = x[nt][u][2] = x[nt][u][3] = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint4 kw[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) kw[t] = *reinterpret_cast<const uint4*>(kt + t * 1024 + (((2 * c + h) ^ g) << 4));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint2 qb[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              qb[nt] = RT == 1 ? q_regs[RT == 1 ? nt * 8 + 4 * h + i : 0] : reinterpret_cast<const uint2*>(gen + V::kQ)[(nt * 8 + 4 * h + i) * 32 + lane];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              uint32_t a[4];
              const uint4 &k0 = kw[2 * u], &k1 = kw[2 * u + 1];
              widen(i == 0 ? k0.x : i == 1 ? k0.y : i == 2 ? k0.z : k0.w, a[0], a[2]);
              widen(i == 0 ? k1.x : i == 1 ? k1.y : i == 2 ? k1.z : k1.w, a[1], a[3]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma_f16_16816(x[nt][u], a[0], a[1], a[2], a[3], qb[nt].x, qb[nt].y);
            }
          }
        }
        // ---- a new reference for the values' scales (rare) ----
        const float vmax = fmaxf(vs0, vs1);
        if (vmax > vref) {
          const float down = vref / vmax;
          vref = vmax;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
              for (int z = 0; z < 4; ++z) acc[nt][j][z] *= down;
        }
        const float inv = 16384.0f / vref, r0 = vs0 * inv, r1 = vs1 * inv;
        float y[RT][4][2];  // [row tile][keys 8 t + g][rows 2c, 2c + 1]
        bool grows = false;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              float v = x[rt * TERMS][t >> 1][2 * (t & 1) + z];
              if (TERMS == 2) v = fmaf(x[rt * TERMS + TERMS - 1][t >> 1][2 * (t & 1) + z], 1.0f / 2048.0f, v);
              y[rt][t][z] = v * (factor[rt][z] * (t < 2 ? ks0 : ks1));
            }
        }
        if (s.cap_l2 > 0.0f) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
              for (int z = 0; z < 2; ++z) y[rt][t][z] = cap_score(y[rt][t][z], s.one_over_cap, s.cap_l2);
        }
        if (masked) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
              for (int z = 0; z < 2; ++z) y[rt][t][z] = kb + 8 * t + g < rows_limit[rt][z] && half != (t < 2 ? 2 : 1) ? y[rt][t][z] : -INFINITY;
        }
        if (s.scores) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              const int r = p.rg * R + rt * 8 + 2 * c + z;  // (single tokens: a row is a query head of the group)
              float* to = s.scores + (static_cast<size_t>(p.e) * s.a.Hq + p.hk * s.G + r) * s.score_row + kb + g;
#pragma unroll
              for (int t = 0; t < 4; ++t)
                if (r < s.G && kb + 8 * t + g < p.limit) to[8 * t] = y[rt][t][z];
            }
        }
        float top[RT][2];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            top[rt][z] = fmaxf(fmaxf(y[rt][0][z], y[rt][1][z]), fmaxf(y[rt][2][z], y[rt][3][z]));
            grows = grows || top[rt][z] > m[rt][z];
          }
        if (__any_sync(0xffffffffu, grows)) {  // (rare once a sequence is under way; one test for all rows leaves straight-line code)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int z = 0; z < 2; ++z) {
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) top[rt][z] = fmaxf(top[rt][z], __shfl_xor_sync(0xffffffffu, top[rt][z], o));
              const float m_new = fmaxf(m[rt][z], top[rt][z]), alpha = ex2(m[rt][z] - (m_new == -INFINITY ? 0.0f : m_new));
              m[rt][z] = m_new;
              l[rt][z] *= alpha;
#pragma unroll
              for (int t = 0; t < TERMS; ++t)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                  acc[rt * TERMS + t][j][z] *= alpha;
                  acc[rt * TERMS + t][j][2 + z] *= alpha;
                }
            }
        }
        uint32_t pb[NT][4];  // B fragments of the values' product, by blocks of eight keys
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
          for (int z = 0; z < 2; ++z) {
            const float from = m[rt][z] == -INFINITY ? 0.0f : m[rt][z];
#pragma unroll
            for (int t = 0; t < 4; ++t) y[rt][t][z] = ex2(y[rt][t][z] - from);
            l[rt][z] += (y[rt][0][z] + y[rt][1][z]) + (y[rt][2][z] + y[rt][3][z]);
#pragma unroll
            for (int t = 0; t < 4; ++t) y[rt][t][z] *= t < 2 ? r0 : r1;
          }
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const uint32_t two = pack_f16x2(y[rt][t][0], y[rt][t][1]);
            pb[rt * TERMS][t] = transposed(two);
            if (TERMS == 2) pb[rt * TERMS + TERMS - 1][t] = transposed(rest_f16x2(two, y[rt][t][0], y[rt][t][1]));
          }
        }
        // ---- values: lane (g, c) reads the dimensions 16 g .. 16 g + 15 of the keys 2c, 2c + 1 of the four blocks; pairs of keys by bytes, then
        // widened, they are the A fragments of eight tiles: dimension 16 g + 2j is row g of tile j, 16 g + 2j + 1 its row g + 8 ----
        uint4 vw[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = 2 * c + (i & 1) + 8 * (i >> 1);
          vw[i] = *reinterpret_cast<const uint4*>(vt + row * 128 + ((g ^ (row & 7)) << 4));
        }
        if (masked) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int key = kb + 2 * c + (i & 1) + 8 * (i >> 1);
            if (key >= p.limit) vw[i] = make_uint4(0u, 0u, 0u, 0u);  // stale rows may hold NaN, and 0 * NaN is NaN
            if (p.sq.len > 1) {
              // a NaN value counts only for the rows that see its key: noted, and put back when the rows are finished
              uint32_t word[4] = {vw[i].x, vw[i].y, vw[i].z, vw[i].w};
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if ((((word[k] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0u)
#pragma unroll
                  for (int b = 0; b < 4; ++b)
                    if ((word[k] >> (8 * b) & 0x7fu) == 0x7fu) {
                      word[k] &= ~(0xffu << (8 * b));
                      atomicMin(&sm_nan[16 * g + 4 * k + b], key);
                    }
              vw[i] = make_uint4(word[0], word[1], word[2], word[3]);
            }
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int kk = 0; kk < 2; ++kk) {
            uint32_t w[4], a[2][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint4& v = vw[4 * kk + i];
              w[i] = k == 0 ? v.x : k == 1 ? v.y : k == 2 ? v.z : v.w;
            }
            widen(__byte_perm(w[0], w[1], 0x5140), a[0][0], a[0][1]);
            widen(__byte_perm(w[2], w[3], 0x5140), a[0][2], a[0][3]);
            widen(__byte_perm(w[0], w[1], 0x7362), a[1][0], a[1][1]);
            widen(__byte_perm(w[2], w[3], 0x7362), a[1][2], a[1][3]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int j = 0; j < 2; ++j)
                mma_f16_16816(acc[nt][2 * k + j], a[j][0], a[j][1], a[j][2], a[j][3], pb[nt][2 * kk], pb[nt][2 * kk + 1]);
          }
      }
      if (half == 1) {  // (the stage once more)
        half = 2;
        continue;
      }
      half = 0;
      __syncwarp();
      load_next();
      sj += kWarps;
      ++count;
    }

    // ---- the warps' sums together, and the rows' results or this CTA's part of them ----
    done += p.end - p.j;
    float* ml = sm_ml + flip * (kWarps * R * 2);  // (a fast warp is at the next piece's while a slow one reads this one's)
    flip ^= 1;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int z = 0; z < 2; ++z) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[rt][z] += __shfl_xor_sync(0xffffffffu, l[rt][z], o);
        if (g == 0) *reinterpret_cast<float2*>(&ml[(warp * R + rt * 8 + 2 * c + z) * 2]) = make_float2(m[rt][z], l[rt][z]);
      }
    __syncthreads();
    // warps 2 and 3 give theirs to 0 and 1: float4 [rt * 8 + 4 z + i][lane] are dimensions 16 g + 4 i .. of row 8 rt + 2 c + z
    float4* merge = reinterpret_cast<float4*>(gen + V::kMerge);
    auto pass = [&](bool add) {
      float4* at = merge + (warp & 1) * (RT * 8 * 32) + lane;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          const float mm = fmaxf(fmaxf(ml[(rt * 8 + 2 * c + z) * 2], ml[(R + rt * 8 + 2 * c + z) * 2]),
                                 fmaxf(ml[(2 * R + rt * 8 + 2 * c + z) * 2], ml[(3 * R + rt * 8 + 2 * c + z) * 2]));
          const float f = ex2(m[rt][z] - (mm == -INFINITY ? 0.0f : mm)) * (vref * (1.0f / 16384.0f));
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float x[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int d = 4 * i + k;
              x[k] = acc[rt * TERMS][d >> 1][2 * (d & 1) + z];
              if (TERMS == 2) x[k] = fmaf(acc[rt * TERMS + TERMS - 1][d >> 1][2 * (d & 1) + z], 1.0f / 2048.0f, x[k]);
            }
            float4& to = at[(rt * 8 + 4 * z + i) * 32];
            const float4 y = add ? to : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            to = make_float4(fmaf(x[0], f, y.x), fmaf(x[1], f, y.y), fmaf(x[2], f, y.z), fmaf(x[3], f, y.w));
          }
        }
    };
    if (warp >= 2) pass(false);
    __syncthreads();
    if (warp < 2) pass(true);
    __syncthreads();
    if (!p.whole && threadIdx.x == 0) {
      Left u{0, 0, 0, p.e, p.hk, p.rg};
      if (shares.cut) {
        u.c0 = part - p.j / shares.cut;
        u.c1 = u.c0 + cuts - 1;
        u.slot0 = 2 * u.c0;
      } else {
        u.c0 = shares.owner(unit_begin);
        u.c1 = shares.owner(unit_begin + p.slices - 1);
        u.slot0 = 2 * u.c0 + (shares.begin(u.c0) == unit_begin ? 0 : 1);
      }
      sm_left[p.first ? 0 : 1] = u;
    }
    const int rows = min(R, p.sq.len * s.G - p.rg * R);
#pragma unroll 1
    for (int r_in = warp; r_in < rows; r_in += kWarps) {  // (a lane: four dimensions)
      const float4* at = merge + ((r_in >> 3) * 8 + 4 * (r_in & 1) + (lane & 3)) * 32 + (lane >> 2) * 4 + ((r_in & 7) >> 1);
      const float4 x0 = at[0], x1 = at[RT * 8 * 32];
      float x[4] = {x0.x + x1.x, x0.y + x1.y, x0.z + x1.z, x0.w + x1.w};
      float2 of[kWarps];
#pragma unroll
      for (int w = 0; w < kWarps; ++w) of[w] = *reinterpret_cast<const float2*>(&ml[(w * R + r_in) * 2]);
      const float mm = fmaxf(fmaxf(of[0].x, of[1].x), fmaxf(of[2].x, of[3].x)), to = mm == -INFINITY ? 0.0f : mm;
      float ll = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) ll = fmaf(of[w].y, ex2(of[w].x - to), ll);
      if (p.sq.len > 1) {
        const int limit = p.sq.pos + (p.rg * R + r_in) / s.G + 1;
#pragma unroll
        for (int d = 0; d < 4; ++d)
          if (limit > sm_nan[4 * lane + d]) x[d] = __uint_as_float(0x7fffffffu);
      }
      const float4 o = make_float4(x[0], x[1], x[2], x[3]);
      if (p.whole) {
        finish_row<T>(s, p.sq, p.hk, p.rg * R + r_in, lane, o, mm, ll);
      } else {
        const size_t slot = (2 * static_cast<size_t>(part) + (p.first ? 0 : 1)) * R + r_in;
        if (lane == 0) *reinterpret_cast<float2*>(s.part_ml + slot * 2) = make_float2(mm, ll);
        *reinterpret_cast<float4*>(s.part_o + slot * 128 + 4 * lane) = o;
      }
    }
    if (done >= share) break;
    unit_begin += p.slices;
    next_piece(s, p, R, share - done);
    ask_row(p);
  }
  if (!ok) {  // (the error word is set and what the call leaves is not a result; copies on their way may still arrive)
    const uint64_t since = global_timer_ns();
    while (global_timer_ns() - since < 2000000ull) __nanosleep(1000);
  }

  // ---- units whose parts this CTA completes ----
  __syncthreads();
  if (threadIdx.x < 2) {
    const Left u = sm_left[threadIdx.x];
    if (u.c1 > u.c0) {
      __threadfence();
      // (the counter goes back to zero with the last arrival)
      if (atomicInc(s.arrivals + u.c0, u.c1 - u.c0) != static_cast<unsigned>(u.c1 - u.c0))
        sm_left[threadIdx.x].c1 = -1;
      __threadfence();
    }
  }
  __syncthreads();
  for (int k = 0; k < 2; ++k) {
    const Left u = sm_left[k];
    const int c0 = u.c0, c1 = u.c1, slot0 = u.slot0;
    if (c1 <= c0) continue;
    const SeqDesc sq = s.seqs[u.e];
    const int rows = min(R, sq.len * s.G - u.rg * R);
    // eight parts at a time: of a row, with more than four rows of two
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
    float4 o[2] = {};
    auto join = [&](int k, float pm, float pl, const float4& x) {
      const float top = fmaxf(m[k], pm), to = top == -INFINITY ? 0.0f : top, a = ex2(m[k] - to), f = ex2(pm - to);
      m[k] = top;
      l[k] = fmaf(pl, f, l[k] * a);
      o[k].x = fmaf(x.x, f, o[k].x * a); o[k].y = fmaf(x.y, f, o[k].y * a); o[k].z = fmaf(x.z, f, o[k].z * a); o[k].w = fmaf(x.w, f, o[k].w * a);
    };
    float2 ml[8];
    float4 x[8];
    auto ask = [&](int i, int q, int r_in) {
      ml[i] = make_float2(-INFINITY, 0.0f);
      x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (q > c1 || r_in >= rows) return;
      const size_t slot = static_cast<size_t>(q == c0 ? slot0 : 2 * q) * R + r_in;
      ml[i] = __ldcg(reinterpret_cast<const float2*>(s.part_ml + slot * 2));
      x[i] = __ldcg(reinterpret_cast<const float4*>(s.part_o + slot * 128 + 4 * lane));
    };
    if (rows > 4) {
#pragma unroll 1
      for (int r0 = warp; r0 < rows; r0 += 2 * kWarps) {
#pragma unroll 1
        for (int q0 = c0; q0 <= c1; q0 += 4) {
#pragma unroll
          for (int i = 0; i < 8; ++i) ask(i, q0 + (i & 3), r0 + (i >> 2) * kWarps);
#pragma unroll
          for (int i = 0; i < 8; ++i) join(i >> 2, ml[i].x, ml[i].y, x[i]);
        }
        finish_row<T>(s, sq, u.hk, u.rg * R + r0, lane, o[0], m[0], l[0]);
        if (r0 + kWarps < rows) finish_row<T>(s, sq, u.hk, u.rg * R + r0 + kWarps, lane, o[1], m[1], l[1]);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          m[i] = -INFINITY;
          l[i] = 0.0f;
          o[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
      }
    } else {
      const int wpr = rows >= 3 ? 1 : rows == 2 ? 2 : 4, r_in = warp / wpr;  // warps for a row
#pragma unroll 1
      for (int q0 = c0 + warp % wpr; q0 <= c1; q0 += 8 * wpr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) ask(i, q0 + i * wpr, r_in);
#pragma unroll
        for (int i = 0; i < 8; ++i) join(0, ml[i].x, ml[i].y, x[i]);
      }
      if (wpr > 1) {
        float4* sm_o = reinterpret_cast<float4*>(gen);  // [warps][32]: the stages are done with
        sm_o[warp * 32 + lane] = o[0];
        if (lane == 0) { sm_ml[2 * warp] = m[0]; sm_ml[2 * warp + 1] = l[0]; }
        __syncthreads();
        if (warp % wpr == 0)
          for (int w = warp + 1; w < warp + wpr; ++w) join(0, sm_ml[2 * w], sm_ml[2 * w + 1], sm_o[w * 32 + lane]);
        __syncthreads();
      }
      if (warp % wpr == 0 && r_in < rows) finish_row<T>(s, sq, u.hk, u.rg * R + r_in, lane, o[0], m[0], l[0]);
    }
  }
}

// Weights of single tokens' calls, from the scores that the attention kernel left: blockIdx = (share of the keys, kv head, entry), four keys a thread.
__global__ void __launch_bounds__(256) cache8_weights_kernel(const __grid_constant__ Shared s) {
  pdl_wait();
  const int e = blockIdx.z, hk = blockIdx.y;
  const SeqDesc sq = s.seqs[e];
  if (!cache8_fits(sq, s.c, s.a.rows, s.max_len)) return;
  float* w = s.c.w + (static_cast<size_t>(sq.slot) * s.c.H + hk) * s.c.cap;
  const float* x = s.scores + (static_cast<size_t>(e) * s.a.Hq + hk * s.G) * s.score_row;
  const float* z = s.lse2 + static_cast<size_t>(sq.row0) * s.a.Hq + hk * s.G;
  for (int j = 4 * (blockIdx.x * 256 + threadIdx.x); j <= sq.pos; j += gridDim.x * 1024) {
    float sum[4] = {}, old[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) old[k] = s.a.decay != 0.0f && j + k <= sq.pos ? w[j + k] : 0.0f;
#pragma unroll 4
    for (int h = 0; h < s.G; ++h) {
      const float4 y = *reinterpret_cast<const float4*>(x + static_cast<size_t>(h) * s.score_row + j);  // (rows of whole fours)
      const float lse = z[h];
      sum[0] += ex2(y.x - lse);
      sum[1] += ex2(y.y - lse);
      sum[2] += ex2(y.z - lse);
      sum[3] += ex2(y.w - lse);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (j + k <= sq.pos) w[j + k] = fmaf(s.a.decay, old[k], sum[k]);
  }
}

// Weights of calls with several tokens: the scores once more, from the rows' lse.  WR of a CTA's eight warps take the same 32 keys of a (kv head, entry),
// each every WR-th eight of the rows, and add their sums through shared memory.
template <typename T>
__global__ void __launch_bounds__(256) cache8_rows_weights_kernel(const __grid_constant__ Shared s, int WR) {
  constexpr int TERMS = sizeof(T) == 4 ? 2 : 1;
  __shared__ float sums[8][32];
  pdl_wait();
  const int e = blockIdx.z, hk = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  const SeqDesc sq = s.seqs[e];
  if (!cache8_fits(sq, s.c, s.a.rows, s.max_len)) return;
  const int live = sq.pos + sq.len, rows = sq.len * s.G, at_once = 8 / WR;
  const size_t head = static_cast<size_t>(sq.slot) * s.c.H + hk;
  for (int first = blockIdx.x * at_once; first * kSlice < live; first += gridDim.x * at_once) {
    const int kb = (first + warp / WR) * kSlice;
    float sum[4] = {};
    if (kb < live) {
      uint32_t ka[2][8][4];  // the keys' A fragments
      float ks[2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int key = kb + 16 * u + 8 * half + g;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int d0 = 16 * (2 * c + h);
            const uint4 w = key < live && d0 < s.c.D ? *reinterpret_cast<const uint4*>(s.c.k + (head * s.c.cap + key) * s.c.D + d0) : make_uint4(0u, 0u, 0u, 0u);
            widen(w.x, ka[u][4 * h][half], ka[u][4 * h][2 + half]);
            widen(w.y, ka[u][4 * h + 1][half], ka[u][4 * h + 1][2 + half]);
            widen(w.z, ka[u][4 * h + 2][half], ka[u][4 * h + 2][2 + half]);
            widen(w.w, ka[u][4 * h + 3][half], ka[u][4 * h + 3][2 + half]);
          }
        }
      ks[0] = s.c.ks[head * s.c.blocks + (kb >> s.c.shift)];
      ks[1] = kb + 16 < live ? s.c.ks[head * s.c.blocks + ((kb + 16) >> s.c.shift)] : 0.0f;
      float raw[32], lse = 0.0f;
      int see = 0;  // keys of the slice that the row sees
      auto ask = [&](int r0) {
        const int r = r0 + g, at = min(r, rows - 1), i = at / s.G, hq = hk * s.G + at - i * s.G;
        const size_t row = static_cast<size_t>(sq.row0) + i;
        load_row(static_cast<const T*>(s.a.q) + row * s.a.ldq + static_cast<size_t>(hq) * s.c.D, s.c.D, r < rows, s.vec_q, c, raw);
        lse = s.lse2[row * s.a.Hq + hq];
        see = r < rows ? sq.pos + i + 1 - kb : 0;
      };
      int r0 = max(0, kb - sq.pos) * s.G / 8 * 8 + 8 * (warp % WR);
      if (r0 < rows) ask(r0);
      for (; r0 < rows; r0 += 8 * WR) {
        uint32_t term[TERMS][16];
        const float f = split_row<TERMS>(raw, s.scale_log2, term);
        float factor[2], z2[2];
        int sees[2];
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          factor[z] = __shfl_sync(0xffffffffu, f, (2 * c + z) * 4);
          z2[z] = __shfl_sync(0xffffffffu, lse, (2 * c + z) * 4);
          sees[z] = __shfl_sync(0xffffffffu, see, (2 * c + z) * 4);
        }
        if (r0 + 8 * WR < rows) ask(r0 + 8 * WR);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float d[TERMS][4] = {};
#pragma unroll
          for (int step = 0; step < 8; ++step)
#pragma unroll
            for (int t = 0; t < TERMS; ++t)
              mma_f16_16816(d[t], ka[u][step][0], ka[u][step][1], ka[u][step][2], ka[u][step][3], term[t][2 * step], term[t][2 * step + 1]);
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int z = 0; z < 2; ++z) {
              float v = d[0][2 * half + z];
              if (TERMS == 2) v = fmaf(d[TERMS - 1][2 * half + z], 1.0f / 2048.0f, v);
              v *= factor[z] * ks[u];
              if (s.cap_l2 > 0.0f) v = cap_score(v, s.one_over_cap, s.cap_l2);
              if (16 * u + 8 * half + g < sees[z]) sum[2 * u + half] += ex2(v - z2[z]);
            }
        }
      }
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      sum[t] += __shfl_xor_sync(0xffffffffu, sum[t], 1);
      sum[t] += __shfl_xor_sync(0xffffffffu, sum[t], 2);
      if (c == 0) sums[warp][8 * t + g] = sum[t];
    }
    __syncthreads();
    if (warp % WR == 0 && kb + lane < live) {
      float all = 0.0f;
      for (int w = 0; w < WR; ++w) all += sums[warp + w][lane];
      float* w = s.c.w + head * s.c.cap + kb + lane;
      *w = s.a.decay == 0.0f ? all : fmaf(s.a.decay, *w, all);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------------ host
struct Plan {
  int kind, rows, parts, groups;
  size_t part_o, part_ml, lse2, scores, widened, bytes;
};
template <typename F>
void for_variant(int kind, F&& f) {  // rows in tiles of eight, or 0 for f32
  if (kind == 0) f(Variant<1, 2>{});
  else if (kind == 1) f(Variant<1, 1>{});
  else if (kind == 2) f(Variant<2, 1>{});
  else if (kind == 3) f(Variant<3, 1>{});
  else f(Variant<4, 1>{});
}
// max_len: of the entries that the main kernel takes.  Scratch has room for either way of dividing a call (see cache8_attention), wherever it lies.
Plan plan_of(const Cache8& c, int f32, int Hq, int rows, int n_seqs, int max_len, int call_len, bool weights) {
  Plan p{};
  auto divide = [&](int len) {
    const long long unit = static_cast<long long>(Hq / c.H) * len;  // rows of the longest entry and a kv head
    // as few passes over the keys as there can be, and no more row tiles than they need
    const long long passes = (unit + 31) / 32;
    p.kind = f32 ? 0 : static_cast<int>((unit + 8 * passes - 1) / (8 * passes));
    for_variant(p.kind, [&](auto v) {
      using V = decltype(v);
      p.rows = V::kRows;
      p.parts = sm_count() * V::kCtas;  // the CTAs that are resident at once
      if (p.parts > TEENY_CACHE8_COUNTER_BYTES / 4) p.parts = TEENY_CACHE8_COUNTER_BYTES / 4;
    });
    p.groups = static_cast<int>((unit + p.rows - 1) / p.rows);
    return static_cast<size_t>(2) * p.parts * p.rows;
  };
  const bool prompts = !f32 && call_len >= cache8_prefill_min_len(c, Hq);
  size_t part_rows = divide(call_len);
  if (prompts) {
    const size_t n = divide(cache8_prefill_min_len(c, Hq) - 1);
    part_rows = part_rows > n ? part_rows : n;
  }
  divide(max_len);
  auto take = [&](size_t n) { const size_t at = p.bytes; p.bytes += (n + 255) / 256 * 256; return at; };
  take(TEENY_CACHE8_COUNTER_BYTES);  // the counters' place is the same for every call, so that calls of any sizes may share scratch
  p.part_o = take(part_rows * 128 * 4);
  p.part_ml = take(part_rows * 2 * 4);
  p.lse2 = weights ? take(static_cast<size_t>(rows) * Hq * 4) : 0;
  p.scores = weights && call_len == 1 ? take(static_cast<size_t>(n_seqs) * Hq * ((c.cap + 3) / 4 * 4) * 4) : 0;
  p.widened = prompts ? take(cache8_prefill_scratch_bytes(c, n_seqs)) : 0;
  return p;
}
int prepare() {
  static std::atomic<unsigned long long> done{0};  // one bit per device; threads may race to set it
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 64 && (done.load(std::memory_order_acquire) >> dev) & 1ull) return 0;
  cudaError_t e = cudaSuccess;
  for (int kind = 0; kind <= 4; ++kind)
    for_variant(kind, [&](auto v) {
      using V = decltype(v);
      const cudaError_t rc = cudaFuncSetAttribute(cache8_attention_kernel<V>, cudaFuncAttributeMaxDynamicSharedMemorySize, V::kBytes);
      if (e == cudaSuccess) e = rc;
    });
  if (e != cudaSuccess) return static_cast<int>(e);
  if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_release);
  return 0;
}
int encode_codes(CUtensorMap* map, const uint8_t* base, int d, const Cache8& c) {
  const uint64_t dims[4] = {static_cast<uint64_t>(d), static_cast<uint64_t>(c.cap), static_cast<uint64_t>(c.H), static_cast<uint64_t>(c.slots)};
  const uint64_t strides[3] = {static_cast<uint64_t>(d), static_cast<uint64_t>(d) * c.cap, static_cast<uint64_t>(d) * c.cap * c.H};
  const uint32_t box[4] = {kCache8Head, kSlice, 1, 1};
  return encode_tensor_map_u8(map, base, 4, dims, strides, box);
}
struct PdlScope {  // kernels of a call behind its first one start their set-up while it ends
  bool was = pdl_enabled();
  PdlScope() { pdl_set_enabled(true); }
  ~PdlScope() { pdl_set_enabled(was); }
};

}  // namespace

size_t cache8_attention_scratch_bytes(const Cache8& c, int f32, int Hq, int rows, int n_seqs, int max_len, bool weights) {
  return plan_of(c, f32, Hq, rows, n_seqs, max_len, max_len, weights).bytes;
}

int cache8_attention(const Cache8& c, const Cache8Attn& a, const SeqDesc* seqs, int n_seqs, int call_len, cudaStream_t st) {
  if (const int rc = prepare()) return rc;
  // Entries of many tokens go to the kernels of cache8_prefill.cu, the others to this file's: by their lengths on the device, which a replayed graph may
  // have changed since the call was captured, so that both are launched wherever an entry can be long.
  const int min_len = cache8_prefill_min_len(c, a.Hq);
  const bool prompts = cache8_prefill_takes(c, a, call_len);
  const int max_len = prompts ? min_len - 1 : call_len;
  const Plan p = plan_of(c, a.f32, a.Hq, a.rows, n_seqs, max_len, call_len, a.weights != 0);
  // the kernels count slices in 32 bits
  if (static_cast<double>(call_len) * (a.Hq / c.H) > 2e9 || static_cast<double>(n_seqs) * c.H * p.groups * ((c.cap + kSlice - 1) / kSlice) > 2e9)
    return TEENY_ERR_BAD_ARG;
  CUtensorMap mk, mv;
  if (const int rc = encode_codes(&mk, c.k, c.D, c)) return rc;
  if (const int rc = encode_codes(&mv, c.v, c.V, c)) return rc;
  Shared s{};
  s.c = c;
  s.a = a;
  s.seqs = seqs;
  s.n_seqs = n_seqs;
  s.max_len = max_len;
  s.score_row = (c.cap + 3) / 4 * 4;
  s.G = a.Hq / c.H;
  s.scale_log2 = a.scale * kLog2e;
  if (a.softcap > 0.0f) {
    s.cap_l2 = a.softcap * kLog2e;
    s.one_over_cap = 1.0f / s.cap_l2;
  }
  uint8_t* scratch = static_cast<uint8_t*>(a.scratch);
  s.arrivals = reinterpret_cast<unsigned*>(scratch);
  s.part_o = reinterpret_cast<float*>(scratch + p.part_o);
  s.part_ml = reinterpret_cast<float*>(scratch + p.part_ml);
  if (a.weights) s.lse2 = reinterpret_cast<float*>(scratch + p.lse2);
  if (a.weights && call_len == 1) s.scores = reinterpret_cast<float*>(scratch + p.scores);
  s.parts = p.parts;
  const int size = a.f32 ? 4 : 2;
  s.vec_q = ((reinterpret_cast<uintptr_t>(a.q) | static_cast<uintptr_t>(a.ldq * size)) & 15) == 0;
  s.vec_o = ((reinterpret_cast<uintptr_t>(a.out) | static_cast<uintptr_t>(a.ldo * size)) & 15) == 0;
  s.err = device_error_word();
  if (!s.err) return TEENY_ERR_DRIVER;
  if (prompts) {
    if (const int rc = cache8_prefill(c, a, s.lse2, scratch + p.widened, seqs, n_seqs, call_len, st)) return rc;
  }
  {
    PdlScope behind;
    if (!prompts) pdl_set_enabled(behind.was);  // (the call's first launch)
    for_variant(p.kind, [&](auto v) {
      using V = decltype(v);
      launch_kernel(cache8_attention_kernel<V>, dim3(p.parts), dim3(32 * kWarps), V::kBytes, st, 1, mk, mv, s);
    });
  }
  if (a.weights) {
    const PdlScope behind;
    // warps for the same keys: as many as share rows usefully
    const long long eights = (static_cast<long long>(s.G) * max_len + 7) / 8;
    const int WR = eights >= 8 ? 8 : eights >= 4 ? 4 : eights >= 2 ? 2 : 1, keys = call_len == 1 ? 1024 : 8 / WR * kSlice;
    const int shares = (c.cap + keys - 1) / keys, most = (4 * sm_count() + n_seqs * c.H - 1) / (n_seqs * c.H);
    const dim3 grid(shares < most ? shares : most, c.H, n_seqs);
    if (call_len == 1) launch_kernel(cache8_weights_kernel, grid, dim3(256), 0, st, 1, s);
    else if (a.f32) launch_kernel(cache8_rows_weights_kernel<float>, grid, dim3(256), 0, st, 1, s, WR);
    else launch_kernel(cache8_rows_weights_kernel<bf16>, grid, dim3(256), 0, st, 1, s, WR);
  }
  return static_cast<int>(cudaGetLastError());
}

}  // namespace teeny
