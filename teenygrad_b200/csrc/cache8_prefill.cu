// Prompts and long portions over the 8-bit cache: their work is the products, not the cache's bytes, so an entry's live tokens are widened to bf16 in
// scratch once (exact: an E4M3 number times a power of two) and the tcgen05 kernel of attention_prefill.cu runs on those.  Widening
// reads one byte and writes two for each number, 0.8 KB a token and kv head at head size 128, against len * group * 512 multiply-adds.
#include <atomic>
#include <type_traits>

#include "common.cuh"
#include "kernels.h"
#include "mma.cuh"

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
// entry's rows see become zeros as well (a masked probability of zero times NaN is NaN) and are noted.  20000 tokens of eight heads, 124 MB: 18 us.
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
  // four 16-byte pieces of codes at a time, straight-line code up to the stores: a piece behind the live tokens reads the last one's place
  const int chunks = kTile * per, last = (live - t0) * per - 1;
  for (int i0 = threadIdx.x; i0 < chunks; i0 += 4 * 256) {
    uint4 w[4];
    float scale[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int i = min(i0 + 256 * m, last), t = t0 + (per == 8 ? i >> 3 : i / per);
      w[m] = src[i];
      scale[m] = scales[t >> c.shift];
    }
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int i = i0 + 256 * m, t = t0 + (per == 8 ? i >> 3 : i / per);
      if (i >= chunks) break;
      uint32_t word[4] = {w[m].x, w[m].y, w[m].z, w[m].w};
      const bool there = i <= last;
      if (of_v && t >= sq.pos) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t is = ((word[k] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;  // bytes 0x7f, 0xff
          nan = nan || (is && there);
          word[k] &= ~((is >> 7) * 0xffu);
        }
      }
      uint4 o[2];
      widen16(make_uint4(word[0], word[1], word[2], word[3]), scale[m], o);
      if (!there) o[0] = o[1] = make_uint4(0u, 0u, 0u, 0u);
      // (whole sectors: as two 16-byte stores a sector is written in halves)
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                   ::"l"(dst + 2 * i), "r"(o[0].x), "r"(o[0].y), "r"(o[0].z), "r"(o[0].w), "r"(o[1].x), "r"(o[1].y), "r"(o[1].z), "r"(o[1].w) : "memory");
    }
  }
  if (of_v) {
    const int any = __syncthreads_or(nan);
    if (threadIdx.x == 0) to.nan[(static_cast<size_t>(blockIdx.z) * c.H + head) * to.tiles + blockIdx.x] = any;
  }
}

// Puts the NaN values back: column d of an output row is NaN from the first token on whose value is NaN there.  blockIdx = (head, entry).
__global__ void __launch_bounds__(128) cache8_nan_kernel(const Cache8 c, const Cache8Attn a, const Widened w, const SeqDesc* seqs, int min_len, int max_len) {
  pdl_wait();
  pdl_trigger();
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

// ---- weights that the cached tokens receive from a prompt's rows ----
// w_j = sum over rows i and the group's query heads of exp2(score_ij - lse2_i): the scores once more, transposed, with keys as the 128 rows of a tcgen05
// product and query rows as its columns, so that a thread has one key and adds along its own registers; no sum crosses threads, and a key
// tile's sums are one CTA's: no atomics.  Bound by the exponentials (128 x 128 of a tile take the special-function units 1024 clocks,
// its product 512; 18000 tiles of five portions: 92 us, 67 of them exponentials).  Two warpgroups take the tiles alternately, over four score buffers in tensor memory.
constexpr int kWThreads = 384, kWQ = 3, kWLse = 4, kWS = 4;
struct WSmem {
  static constexpr int kK = 0;                                // two key tiles, two boxes of [128][64] each
  static constexpr int kQ = kK + 2 * 32768;                   // ring of query tiles
  static constexpr int kLse = kQ + kWQ * 32768;               // f32 [kWLse][128], negated
  static constexpr int kSum = kLse + kWLse * 512;             // f32 [2][128]: what the second warpgroup hands over, by item
  static constexpr int kBar = kSum + 2 * 512;
  static constexpr int kTotal = kBar + 256 + 1024;
};
struct WeightsArgs {
  Cache8 c;
  const SeqDesc* seqs;
  const float* lse2;  // [rows][Hq]
  int n_seqs, key_rows, tiles, min_len, max_len, rows, Hq;
  float scale_log2, one_over_cap, cap_l2, decay;
  int* err;
};

template <bool CAP>
__global__ void __launch_bounds__(kWThreads, 1)
cache8_prompt_weights_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ WeightsArgs a) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* gen = smem_raw + (base - smem_u32(smem_raw));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int K_FULL = 0, K_EMPTY = 2, Q_FULL = 4, Q_EMPTY = Q_FULL + kWQ, S_FULL = Q_EMPTY + kWQ, S_EMPTY = S_FULL + kWS, L_FULL = S_EMPTY + kWS,
                L_EMPTY = L_FULL + kWLse, X_FULL = L_EMPTY + kWLse, X_EMPTY = X_FULL + 2, kBars = X_EMPTY + 2;
  static_assert(8 * kBars + 4 <= 256, "barrier block");
  auto bar = [&](int i) { return base + WSmem::kBar + 8u * i; };
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gen + WSmem::kBar + 8 * kBars);
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_q);
    for (int i = 0; i < kBars; ++i)
      mbar_init(bar(i), (i >= S_EMPTY && i < L_FULL) || i >= L_EMPTY ? 128 : i >= L_FULL ? 32 : 1);
    mbar_fence_init();
  }
  if (warp == 3) {
    tmem_alloc(base + WSmem::kBar + 8 * kBars, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  pdl_wait();
  const int G = a.Hq / a.c.H, per_tile = a.n_seqs * a.c.H;
  // item(n, entry, sq, kv head, first key, first query tile, query tiles) for every key tile of this CTA; key tiles with most rows come first
  auto walk = [&](auto&& item) {
    int n = 0;
    for (int i = blockIdx.x; i < per_tile * a.tiles; i += gridDim.x) {
      const int kt = i / per_tile, e = i % per_tile / a.c.H, hk = i % a.c.H;
      const SeqDesc sq = a.seqs[e];
      if (sq.len < a.min_len || !cache8_fits(sq, a.c, a.rows, a.max_len) || kt * 128 >= sq.pos + sq.len) continue;
      if (!item(n++, e, sq, hk, kt * 128, max(0, kt * 128 - sq.pos) / 128, (sq.len + 127) / 128)) return;
    }
  };
  if (warp == 0) {
    if (lane == 0) {
      int t = 0;
      walk([&](int n, int e, const SeqDesc& sq, int hk, int key0, int q0, int q1) {
        const int kb = n & 1;
        if (!mbar_wait(bar(K_EMPTY + kb), (n >> 1 & 1) ^ 1, a.err, DEVERR_ATTN_PRODUCER)) return false;
        mbar_expect_tx(bar(K_FULL + kb), 32768);
        for (int x = 0; x < 2; ++x) tma_load_3d(base + WSmem::kK + kb * 32768 + x * 16384, &tmap_k, bar(K_FULL + kb), 64 * x, e * a.key_rows + key0, hk);
        for (int g = 0; g < G; ++g)
          for (int q = q0; q < q1; ++q, ++t) {
            const int st = t % kWQ;
            if (!mbar_wait(bar(Q_EMPTY + st), (t / kWQ & 1) ^ 1, a.err, DEVERR_ATTN_PRODUCER)) return false;
            mbar_expect_tx(bar(Q_FULL + st), 32768);
            for (int x = 0; x < 2; ++x)
              tma_load_3d(base + WSmem::kQ + st * 32768 + x * 16384, &tmap_q, bar(Q_FULL + st), 64 * x, sq.row0 + q * 128, hk * G + g);
          }
        return true;
      });
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = make_idesc_bf16(128, 128, false, false);
      const uint64_t kd = make_smem_desc_sw128(base + WSmem::kK, 16, 1024), qd = make_smem_desc_sw128(base + WSmem::kQ, 16, 1024);
      int t = 0;
      walk([&](int n, int, const SeqDesc&, int, int, int q0, int q1) {
        const int kb = n & 1, tiles = G * (q1 - q0);
        if (!mbar_wait(bar(K_FULL + kb), n >> 1 & 1, a.err, DEVERR_ATTN_MMA)) return false;
        for (int i = 0; i < tiles; ++i, ++t) {
          const int st = t % kWQ, sb = t % kWS;
          if (!mbar_wait(bar(Q_FULL + st), t / kWQ & 1, a.err, DEVERR_ATTN_MMA)) return false;
          if (!mbar_wait(bar(S_EMPTY + sb), (t / kWS & 1) ^ 1, a.err, DEVERR_ATTN_MMA)) return false;
          tc_fence_after();
          const uint64_t ka = kd + static_cast<uint64_t>(kb * (32768 >> 4)), qb = qd + static_cast<uint64_t>(st * (32768 >> 4));
          umma_bf16_ss_x4<2, 2>(tmem + sb * 128, ka, qb, idesc, 0u);
          umma_bf16_ss_x4<2, 2>(tmem + sb * 128, ka + (16384 >> 4), qb + (16384 >> 4), idesc, 1u);
          umma_commit(bar(Q_EMPTY + st));
          umma_commit(bar(S_FULL + sb));
        }
        umma_commit(bar(K_EMPTY + kb));
        return true;
      });
    }
  } else if (warp == 2) {
    int t = 0;
    walk([&](int, int, const SeqDesc& sq, int hk, int, int q0, int q1) {
      for (int g = 0; g < G; ++g)
        for (int q = q0; q < q1; ++q, ++t) {
          const int sl = t % kWLse;
          if (!mbar_wait(bar(L_EMPTY + sl), (t / kWLse & 1) ^ 1, a.err, DEVERR_ATTN_PRODUCER)) return false;
          float* to = reinterpret_cast<float*>(gen + WSmem::kLse) + sl * 128;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int i = q * 128 + x * 32 + lane;
            to[x * 32 + lane] = i < sq.len ? -a.lse2[(static_cast<size_t>(sq.row0) + i) * a.Hq + hk * G + g] : 0.0f;
          }
          mbar_arrive(bar(L_FULL + sl));
        }
      return true;
    });
  } else if (warp >= 4) {
    const int wg = (warp - 4) >> 2, quarter = warp & 3, key = quarter * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const float2 sc2 = make_float2(a.scale_log2, a.scale_log2);
    int t = 0, last_n = -1;
    float *last_w = nullptr, last_sum = 0.0f;  // the first warpgroup's last item, but for the other's part
    auto finish = [&](int n) {
      if (!mbar_wait(bar(X_FULL + (n & 1)), n >> 1 & 1, a.err, DEVERR_ATTN_SOFTMAX)) return false;
      const float other = reinterpret_cast<const float*>(gen + WSmem::kSum)[(n & 1) * 128 + key];
      mbar_arrive(bar(X_EMPTY + (n & 1)));
      if (last_w) *last_w = last_sum + other;
      return true;
    };
    walk([&](int n, int, const SeqDesc& sq, int hk, int key0, int q0, int q1) {
      const bool mine = key0 + key < sq.pos + sq.len;
      float* w = a.c.w + (static_cast<size_t>(sq.slot) * a.c.H + hk) * a.c.cap + key0 + key;
      const float old = wg == 0 && mine && a.decay != 0.0f ? *w : 0.0f;
      float2 sum[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
      for (int g = 0; g < G; ++g)
        for (int q = q0; q < q1; ++q, ++t) {
          if ((t & 1) != wg) continue;
          const int sb = t % kWS, sl = t % kWLse;
          if (!mbar_wait(bar(L_FULL + sl), t / kWLse & 1, a.err, DEVERR_ATTN_SOFTMAX)) return false;
          if (!mbar_wait(bar(S_FULL + sb), t / kWS & 1, a.err, DEVERR_ATTN_SOFTMAX)) return false;
          tc_fence_after();
          const int hidden = key0 + key - sq.pos - q * 128;  // columns before this one do not see the key
          const int rows = sq.len - q * 128;  // columns from this one on are not the entry's
          const bool masked = key0 + 127 > sq.pos + q * 128 || rows < 128;
          const float4* lse = reinterpret_cast<const float4*>(gen + WSmem::kLse + sl * 512);
          // (the masked tiles have a loop of their own: a test at every element kept the others' from being worked on side by side)
          auto add = [&](auto with_mask) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              uint32_t r[32];
              tmem_ld_32x32(tmem + lane_addr + sb * 128 + x * 32, r);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const float4 z = lse[x * 8 + i];
                float2 p[2] = {make_float2(__uint_as_float(r[4 * i]), __uint_as_float(r[4 * i + 1])), make_float2(__uint_as_float(r[4 * i + 2]), __uint_as_float(r[4 * i + 3]))};
                const float2 minus[2] = {make_float2(z.x, z.y), make_float2(z.z, z.w)};
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                  if (CAP) {
                    p[k].x = cap_score(p[k].x * a.scale_log2, a.one_over_cap, a.cap_l2);
                    p[k].y = cap_score(p[k].y * a.scale_log2, a.one_over_cap, a.cap_l2);
                    p[k] = __fadd2_rn(p[k], minus[k]);
                  } else {
                    p[k] = __ffma2_rn(p[k], sc2, minus[k]);
                  }
                  if (with_mask.value) {
                    const int col = x * 32 + 4 * i + 2 * k;
                    if (col < hidden || col >= rows) p[k].x = -INFINITY;
                    if (col + 1 < hidden || col + 1 >= rows) p[k].y = -INFINITY;
                  }
                  sum[k] = __fadd2_rn(sum[k], make_float2(ex2(p[k].x), ex2(p[k].y)));
                }
              }
            }
          };
          if (masked) add(std::true_type{});
          else add(std::false_type{});
          tc_fence_before();
          mbar_arrive(bar(S_EMPTY + sb));
          mbar_arrive(bar(L_EMPTY + sl));
        }
      // the second warpgroup's part to the first, which adds it an item later: by then it is there
      const float total = (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      if (wg == 1) {
        if (!mbar_wait(bar(X_EMPTY + (n & 1)), (n >> 1 & 1) ^ 1, a.err, DEVERR_ATTN_SOFTMAX)) return false;
        reinterpret_cast<float*>(gen + WSmem::kSum)[(n & 1) * 128 + key] = total;
        mbar_arrive(bar(X_FULL + (n & 1)));
        return true;
      }
      if (n > 0 && !finish(n - 1)) return false;
      last_w = mine ? w : nullptr;
      last_sum = fmaf(a.decay, old, total);
      last_n = n;
      return true;
    });
    if (wg == 0 && last_n >= 0) finish(last_n);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 3) {
    if (*reinterpret_cast<volatile int*>(a.err) != 0) {  // (products under way may still write there)
      const uint64_t t0 = global_timer_ns();
      while (global_timer_ns() - t0 < 2000000ull) __nanosleep(1000);
    }
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

int prompt_weights(const Cache8& c, const Cache8Attn& a, const Widened& w, const float* lse2, const SeqDesc* seqs, int min_len, int max_len, cudaStream_t st) {
  static std::atomic<unsigned long long> done{0};  // one bit per device; threads may race to set it
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !((done.load(std::memory_order_acquire) >> dev) & 1ull)) {
    cudaError_t e = cudaFuncSetAttribute(cache8_prompt_weights_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, WSmem::kTotal);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(cache8_prompt_weights_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, WSmem::kTotal);
    if (e != cudaSuccess) return static_cast<int>(e);
    if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_release);
  }
  const uint64_t keys = static_cast<uint64_t>(w.n_seqs) * w.key_rows, D = c.D;
  const uint32_t box[3] = {64, 128, 1};
  CUtensorMap mk, mq;
  const uint64_t kdims[3] = {D, keys, static_cast<uint64_t>(c.H)}, kstrides[2] = {D * 2, D * 2 * keys};
  const uint64_t qdims[3] = {D, static_cast<uint64_t>(a.rows), static_cast<uint64_t>(a.Hq)}, qstrides[2] = {static_cast<uint64_t>(a.ldq) * 2, D * 2};
  if (const int rc = encode_tensor_map_bf16(&mk, w.k, 3, kdims, kstrides, box)) return rc;
  if (const int rc = encode_tensor_map_bf16(&mq, a.q, 3, qdims, qstrides, box)) return rc;
  WeightsArgs t{};
  t.c = c;
  t.seqs = seqs;
  t.lse2 = lse2;
  t.n_seqs = w.n_seqs;
  t.key_rows = w.key_rows;
  t.tiles = w.tiles;
  t.min_len = min_len;
  t.max_len = max_len;
  t.rows = a.rows;
  t.Hq = a.Hq;
  t.scale_log2 = a.scale * 1.4426950408889634f;
  if (a.softcap > 0.0f) {
    t.cap_l2 = a.softcap * 1.4426950408889634f;
    t.one_over_cap = 1.0f / t.cap_l2;
  }
  t.decay = a.decay;
  t.err = device_error_word();
  if (!t.err) return TEENY_ERR_DRIVER;
  const long long items = static_cast<long long>(w.tiles) * w.n_seqs * c.H, sms = sm_count();
  launch_kernel(a.softcap > 0.0f ? cache8_prompt_weights_kernel<true> : cache8_prompt_weights_kernel<false>, dim3(static_cast<unsigned>(items < sms ? items : sms)), dim3(kWThreads), WSmem::kTotal, st, 1, mk, mq, t);
  return static_cast<int>(cudaGetLastError());
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
         a.scale < 1e30f && (a.softcap == 0.0f || a.scale / a.softcap < 1e30f);
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
    int rc = attention_prefill_ragged(c, a, w.k, w.v, w.key_rows, lse2, seqs + e, w.n_seqs, min_len, max_len, st);
    if (rc == 0 && a.weights) rc = prompt_weights(c, a, w, lse2, seqs + e, min_len, max_len, st);
    if (rc == 0) launch_kernel(cache8_nan_kernel, dim3(c.H, w.n_seqs), dim3(128), 0, st, 1, c, a, w, seqs + e, min_len, max_len);
    pdl_set_enabled(pdl);
    if (rc) return rc;
  }
  return static_cast<int>(cudaGetLastError());
}

}  // namespace teeny
