// W8A8 products for sm_100a: out[m, n] = (sum_k A8[m, k] W8[n, k]) * a_scale[m]
// * w_scale[n] (+ bias[n]), and their gated form act(gate) * up.
//
// int8 runs tcgen05 kind::i8 (int32 accumulators: exact), e4m3 runs
// kind::f8f6f4 (fp32). Both operands are K-major rows, which is how TMA stages
// them (128-byte swizzled tiles of 128 bytes of K) and the tensor core reads
// them: no transposition, no conversion, no pass through registers. The
// epilogue applies the scales in fp32 and rounds once to the output's type.
//
// Two kernels:
//  * w8a8_swap_kernel, few tokens: the weights are the MMA's 128-row operand,
//    the tokens its 16..256 columns (just as many as needed), one tile per CTA.
//    The product is a weight stream there (16 x 28672 x 8192: 38 us = 6.2 TB/s);
//    K is split over a thread-block cluster when there are too few column tiles
//    to keep every SM loading, and the partial sums meet in distributed shared
//    memory (in rank order; no workspace, no atomics). A CTA gives its tensor
//    memory back before it waits for the others of its cluster.
//  * w8a8_pair_kernel, many tokens: persistent, 256 x 256 tiles of a CTA pair
//    (cta_group::2), two accumulators so that a tile's epilogue overlaps the
//    next one's main loop (4096 x 11008 x 4096 int8: 117 us = 3.2 POP/s, the
//    tensor cores' rate; held for seconds the power cap makes it 141). Gated: CTA 0 stages 128 gate channels and CTA 1 the
//    same 128 up channels, so one MMA makes both halves and a row's epilogue
//    thread holds gate and up of each of its 128 outputs.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "pk_common.cuh"

namespace pk {
namespace {

constexpr int kBK = 128;  // bytes of K per stage: one swizzle row
constexpr int kKSteps = kBK / 32;
constexpr int kTmaWarp = 0, kMmaWarp = 1, kEpiWarp0 = 2;
constexpr int kEpiWarps = 8;  // two per TMEM lane quarter, half the columns each
constexpr int kEpiThreads = kEpiWarps * 32;
constexpr int kThreads = kEpiWarp0 * 32 + kEpiThreads;

struct Params {
  const float* a_scale;
  const float* w_scale[2];
  const float* bias;
  void* out;
  int64_t ldo;
  int M, N, K;
  int out_dtype, act;
  int rows16;        // the output's rows start on 16-byte boundaries
  // swap: CTAs per tile along K (the cluster), tokens of a tile (a multiple of
  // 16), the ring, TMEM columns, whether a split's sums have memory beside the ring
  int split, nt, stages, stage_bytes, tmem_cols, own_red;
  int pieces;        // swap: accumulators that a CTA's K range is summed in
  int num_m, num_n;  // tiles
  // pair: units that are whole tiles; each later tile is `parts` narrower units
  int whole, parts;
  int box;           // pair: channels of a TMA box (32 where there are quarter units, else 64)
  int* status;
};

// kind::i8: D int32 (format 2), operands signed (1); kind::f8f6f4: D fp32, e4m3 (0)
constexpr uint32_t idesc8(bool e4m3, int m, int n) {
  return (e4m3 ? 1u << 4 : (2u << 4) | (1u << 7) | (1u << 10)) |
         (static_cast<uint32_t>(n) >> 3 << 17) | (static_cast<uint32_t>(m) >> 4 << 24);
}

// One lane of a converged warp. The MMA warps run their loops with all lanes and
// issue under this predicate: in a loop of one lane every operand of a
// tcgen05.mma went from a vector to a uniform register, and a K tile's four MMAs
// took ~550 cycles to issue, whatever their size.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}

// After a wait that ran out: time (~100 us) for the copies and MMAs already
// issued to end before the CTA's shared and tensor memory are released.
__device__ __noinline__ void drain() {
  const long long t0 = clock64();
  while (clock64() - t0 < 200000) __nanosleep(1000);
}

template <bool kE4M3>
__device__ __forceinline__ void umma8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                      uint32_t acc) {
  if constexpr (kE4M3) {
    umma_f8(d, a, b, idesc, acc);
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
  }
}

template <bool kE4M3>
__device__ __forceinline__ void umma8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                           uint32_t acc) {
  if constexpr (kE4M3) {
    umma_f8_pair(d, a, b, idesc, acc);
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
  }
}

// Named barrier over `nthreads` threads that tells each whether any said true.
__device__ __forceinline__ bool named_bar_or(int id, int nthreads, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %3, 0;\n\t"
      "barrier.cta.red.or.aligned.pred q, %1, %2, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(nthreads), "r"(static_cast<uint32_t>(v))
      : "memory");
  return r != 0;
}

template <bool kE4M3>
__device__ __forceinline__ float acc_value(uint32_t raw) {
  return kE4M3 ? __uint_as_float(raw) : static_cast<float>(static_cast<int>(raw));
}

// g * sigmoid(t): SiLU with t = g; GELU's tanh form with t = 2 sqrt(2/pi) (g +
// 0.044715 g^3), since (1 + tanh(t/2)) / 2 = sigmoid(t). The fast exponential
// and quotient are off by about |t| + 6 last places where t < 0 (in the tail,
// where the result vanishes) and by a few elsewhere; expf and an IEEE division
// made the epilogue of a 256 x 128 tile longer than its main loop (4096 x 11008
// x 4096: 362 us).
__device__ __forceinline__ float gated(float g, float u, int act) {
  const float t = act == PK_ACT_SILU ? g : 1.5957691216057308f * (g + 0.044715f * g * g * g);
  return __fdividef(g, 1.0f + __expf(-t)) * u;
}

__device__ __forceinline__ void put(float* o, float v) { *o = v; }
__device__ __forceinline__ void put(__half* o, float v) { *o = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* o, float v) { *o = __float2bfloat16_rn(v); }

__device__ __forceinline__ void store_one(void* out, int dtype, int64_t i, float v) {
  if (dtype == PK_F16)
    put(static_cast<__half*>(out) + i, v);
  else
    store_elem(out, dtype, i, v);
}

// f(the output as its own type)
template <typename F>
__device__ __forceinline__ void with_type(void* out, int dtype, F f) {
  if (dtype == PK_F32) f(static_cast<float*>(out));
  else if (dtype == PK_BF16) f(static_cast<__nv_bfloat16*>(out));
  else f(static_cast<__half*>(out));
}

__device__ __forceinline__ void lds_floats(uint32_t addr, float (&v)[4]) {
  const uint4 u = lds_v4(addr);
  v[0] = __uint_as_float(u.x);
  v[1] = __uint_as_float(u.y);
  v[2] = __uint_as_float(u.z);
  v[3] = __uint_as_float(u.w);
}

__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// Two outputs as one word of a 16-bit type.
__device__ __forceinline__ uint32_t pack16(int dtype, float a, float b) {
  if (dtype == PK_BF16) {
    const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&p);
  }
  const __half2 p = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&p);
}

// ---------------------------------------------------------------------------
// Few tokens: D[channel, token], one tile of 128 channels x nt tokens per CTA.
// ---------------------------------------------------------------------------
constexpr int kWTile = 128 * kBK;  // 16 KB: one stage of 128 channels
constexpr int kMaxTokens = 256;    // tokens of a tile: the MMA's columns

constexpr int kMaxSplit = 8;
constexpr int kSwapBars = 256;      // bytes for its barriers (at most 15 stages)

template <bool kE4M3, bool kGated>
__global__ void __launch_bounds__(kThreads)
    w8a8_swap_kernel(const __grid_constant__ CUtensorMap tmA,
                     const __grid_constant__ CUtensorMap tmW0,
                     const __grid_constant__ CUtensorMap tmW1, const Params p) {
  constexpr int kW = kGated ? 2 : 1;  // weight tiles per stage
  const int nt = p.nt, stages = p.stages, stage_bytes = p.stage_bytes;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  // after the ring: token scales, barriers, and (own_red) the sums of a K split
  float* s_sa = reinterpret_cast<float*>(smem + stages * stage_bytes);
  uint64_t* full = reinterpret_cast<uint64_t*>(s_sa + kMaxTokens);
  uint64_t* empty = full + stages;
  uint64_t* done = empty + stages;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(done + 1);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // split fastest (the cluster), then the token tiles that share a weight tile
  const int ks = static_cast<int>(blockIdx.x % p.split);
  const int tile = static_cast<int>(blockIdx.x / p.split);
  const int m0 = (tile % p.num_m) * nt, n0 = (tile / p.num_m) * 128;
  const int k_tiles = (p.K + kBK - 1) / kBK;
  const int kt0 = static_cast<int>(static_cast<int64_t>(ks) * k_tiles / p.split);
  const int kt1 = static_cast<int>(static_cast<int64_t>(ks + 1) * k_tiles / p.split);

  if (warp == kTmaWarp && lane == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(done, 1);
    fence_barrier_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmW0);
    if (kGated) tma_prefetch_desc(&tmW1);
    // the first weights start towards L2 while the previous kernel ends (a
    // hint: nothing is read that it may still write)
    for (int kt = kt0; kt < kt1 && kt < kt0 + stages; ++kt) {
      tma_prefetch_l2_2d(&tmW0, kt * kBK, n0);
      if (kGated) tma_prefetch_l2_2d(&tmW1, kt * kBK, n0);
    }
  }
  // Memory beside the ring takes sums from CTAs that know of its owner's start. The
  // word goes out before the wait for tensor memory, so that whoever holds some
  // waits for nothing but its own loads and MMAs: clusters of several streams that
  // share SMs then cannot hold on one of them what the other needs on the next.
  __syncwarp();
  if (p.own_red) cluster_arrive_unordered();
  if (warp == kMmaWarp) tmem_alloc(tmem_holder, p.tmem_cols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  griddep_wait();
  griddep_launch_dependents();

  bool fail = false;
  if (warp == kTmaWarp) {
    uint8_t* base = smem;
    uint64_t* bar = full;
    uint32_t parity = 1;  // a fresh barrier's previous phase: the first round does not wait
    for (int kt = kt0; kt < kt1; ++kt) {
      fail = __any_sync(0xffffffffu, !mbar_wait(bar + stages, parity, p.status, kSiteW8SwapProducer));
      if (fail) break;
      if (elect_one()) {
        mbar_arrive_expect_tx(bar, stage_bytes);
        tma_load_2d(base, &tmW0, bar, kt * kBK, n0);
        if (kGated) tma_load_2d(base + kWTile, &tmW1, bar, kt * kBK, n0);
        tma_load_2d(base + kW * kWTile, &tmA, bar, kt * kBK, m0);
      }
      __syncwarp();
      base += stage_bytes;
      if (++bar == empty) {
        bar = full;
        base = smem;
        parity ^= 1;
      }
    }
  } else if (warp == kMmaWarp) {
    const uint32_t idesc = idesc8(kE4M3, 128, nt);
    const uint64_t desc0 = make_smem_desc(0, 16, 1024);  // a tile at address 0
    uint32_t w_base = smem_u32(smem), parity = 0, d_tmem = tmem;
    const int per_piece = (kt1 - kt0 + p.pieces - 1) / p.pieces;
    int in_piece = 0;  // K tiles in the current accumulator
    uint64_t* bar = full;
    for (int kt = kt0; kt < kt1; ++kt) {
      // a warp gives up as one
      fail = __any_sync(0xffffffffu, !mbar_wait(bar, parity, p.status, kSiteW8SwapMma));
      if (fail) break;
      if (elect_one()) {
        const uint64_t wd = desc0 + (w_base >> 4), ad = wd + (kW * kWTile >> 4);
#pragma unroll
        for (int s = 0; s < kKSteps; ++s) {
#pragma unroll
          for (int w = 0; w < kW; ++w)
            umma8<kE4M3>(d_tmem + w * nt, wd + ((w * kWTile + s * 32) >> 4), ad + (s * 32 >> 4),
                         idesc, s > 0 || in_piece > 0 ? 1u : 0u);
        }
        umma_commit(bar + stages);
        if (kt + 1 == kt1) umma_commit(done);
      }
      __syncwarp();
      if (++in_piece == per_piece) {
        in_piece = 0;
        d_tmem += kW * nt;
      }
      w_base += stage_bytes;
      if (++bar == empty) {
        bar = full;
        w_base = smem_u32(smem);
        parity ^= 1;
      }
    }
  }

  // ---- epilogue: a thread holds one channel, the columns are tokens ----
  const int q = warp & 3;  // TMEM lane quarter this warp may access
  const int nl = q * 32 + lane;
  const int tokens = min(nt, p.M - m0);
  const bool epi = warp >= kEpiWarp0;
  const int part = (warp - kEpiWarp0) >> 2;  // which half of the tokens (epilogue warps)
  const uint32_t sa_addr = smem_u32(s_sa);
  const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16);
  // eight accumulator columns, the pieces of K added up (used when the loads of
  // a caller's tmem_ld_wait are in)
  const int used = (kt1 - kt0 + p.pieces - 1) / p.pieces;
  const int filled = (kt1 - kt0 + used - 1) / used;
  auto load_sums = [&](int col, uint32_t (&x)[8]) {
    tmem_ld_32x32b_x8(taddr + col, x);
    if (kE4M3 && filled > 1) {
      for (int i = 1; i < filled; ++i) {
        uint32_t y[8];
        tmem_ld_32x32b_x8(taddr + i * kW * nt + col, y);
        tmem_ld_wait();
#pragma unroll
        for (int e = 0; e < 8; ++e)
          x[e] = __float_as_uint(__uint_as_float(x[e]) + __uint_as_float(y[e]));
      }
    }
  };
  // this thread's channel and what its epilogue multiplies and adds
  const int et = tid - kEpiWarp0 * 32;
  const int ch = p.split == 1 ? nl : et & 127;
  const int n = n0 + ch;
  const bool inside = epi && n < p.N;
  const bool biased = !kGated && p.bias != nullptr;
  float sw[kW], bias = 0.0f;
  auto finish = [&](float sa, float x, float y) {
    x = x * sa * sw[0];
    if constexpr (kGated) return gated(x, y * sa * sw[kW - 1], p.act);
    return biased ? x + bias : x;
  };
  if (epi) {
#pragma unroll
    for (int w = 0; w < kW; ++w) sw[w] = inside ? p.w_scale[w][n] : 0.0f;
    if (biased && inside) bias = p.bias[n];
    for (int m = et; m < tokens; m += kEpiThreads) s_sa[m] = p.a_scale[m0 + m];
    named_bar_sync(1, kEpiThreads);
    // a warp gives up as one (its TMEM loads are collective)
    fail = __any_sync(0xffffffffu, !mbar_wait(done, 0, p.status, kSiteW8SwapEpilogue));
    tc_fence_after();
  }
  if (p.split == 1) {
    if (epi && !fail) {
      with_type(p.out, p.out_dtype, [&](auto* out) {
        // Eight tokens at a time: everything is read and computed before the
        // first store, which the compiler must otherwise keep the next token's
        // scale behind (110 cycles an output: 256 tokens took 7 us).
#pragma unroll 1
        for (int c = part * (nt / 2); c < (part + 1) * (nt / 2) && c < tokens; c += 8) {
          uint32_t x[8], y[8];
          load_sums(c, x);
          if (kGated) load_sums(nt + c, y);
          const uint4 s0 = lds_v4(sa_addr + c * 4), s1 = lds_v4(sa_addr + c * 4 + 16);
          const uint32_t sa[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
          tmem_ld_wait();
          float v[8];
#pragma unroll
          for (int i = 0; i < 8; ++i)
            v[i] = finish(__uint_as_float(sa[i]), acc_value<kE4M3>(x[i]),
                          kGated ? acc_value<kE4M3>(y[i]) : 0.0f);
          auto* o = out + static_cast<int64_t>(m0 + c) * p.ldo + n;
#pragma unroll
          for (int i = 0; i < 8; ++i, o += p.ldo)
            if (inside && c + i < tokens) put(o, v[i]);
        }
      });
    }
  } else {
    // Rank r of the cluster owns tokens [r * per, (r + 1) * per) and adds the ranks'
    // sums of them in order. Sums that have memory beside the ring are stored into
    // the owner's, more of them into this CTA's own drained ring, from where their
    // owner fetches them.
    const int per = (tokens + p.split - 1) / p.split;
    const uint32_t red = smem_u32(
        p.own_red ? smem + stages * stage_bytes + kMaxTokens * 4 + kSwapBars : smem);
    __syncwarp();
    if (p.own_red) cluster_wait();
    if (epi && !fail) {
#pragma unroll 1
      for (int c = part * (nt / 2); c < (part + 1) * (nt / 2) && c < tokens; c += 8) {
#pragma unroll
        for (int w = 0; w < kW; ++w) {
          uint32_t x[8];
          load_sums(w * nt + c, x);
          tmem_ld_wait();
          if (!p.own_red) {  // [token][weight][channel]
#pragma unroll
            for (int i = 0; i < 8; ++i)
              sts_f32(red + ((c + i) * kW + w) * 512 + nl * 4, __uint_as_float(x[i]));
            continue;
          }
          int owner = c / per, at = c - owner * per;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if (c + i < tokens) {
              // [token of the owner][weight][source rank][channel]
              const uint32_t to = red + ((at * kW + w) * p.split + ks) * 512 + nl * 4;
              st_cluster_u32(cluster_map(to, owner), x[i]);
              if (++at == per) {
                at = 0;
                ++owner;
              }
            }
          }
        }
      }
    }
    // the sums are where they are read; this CTA's tensor memory goes back before it
    // waits for the others
    __syncwarp();
    cluster_arrive();
    tc_fence_before();
    fail = __syncthreads_or(fail);
    if (fail) drain();
    tc_fence_after();
    if (warp == kMmaWarp) tmem_dealloc(tmem, p.tmem_cols);
    __syncwarp();
    const int first = ks * per, last = min(first + per, tokens);
    auto add = [&](float a, float b) {
      return kE4M3 ? a + b : __uint_as_float(__float_as_uint(a) + __float_as_uint(b));
    };
    auto value = [&](float sum) { return acc_value<kE4M3>(__float_as_uint(sum)); };
    if (p.own_red) {
      cluster_wait();
      if (!epi || fail) return;
      auto total = [&](int m, int w) {
        const uint32_t at = red + (((m - first) * kW + w) * p.split) * 512 + ch * 4;
        float v = lds_f32(at);
#pragma unroll
        for (int j = 1; j < kMaxSplit; ++j)
          if (j < p.split) v = add(v, lds_f32(at + j * 512));
        return value(v);
      };
      with_type(p.out, p.out_dtype, [&](auto* out) {
        // four tokens (of this thread's parity) at a time, read before stored
#pragma unroll 1
        for (int m = first + (et >> 7); m < last; m += 8) {
          float v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int mm = min(m + 2 * i, last - 1);
            v[i] = finish(lds_f32(sa_addr + mm * 4), total(mm, 0),
                          kGated ? total(mm, kW - 1) : 0.0f);
          }
          auto* o = out + static_cast<int64_t>(m0 + m) * p.ldo + n;
#pragma unroll
          for (int i = 0; i < 4; ++i, o += 2 * p.ldo)
            if (inside && m + 2 * i < last) put(o, v[i]);
        }
      });
      return;
    }
    // Four channels a thread, eight tokens at a time: every rank's sums of a token on
    // their way before the first is added (128 x 4096 x 4096 9.4 us, by single words
    // 13.5).
    const int c4 = (et & 31) * 4, n4 = n0 + c4;
    float s4[kW][4], b4[4];
    if (epi) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
#pragma unroll
        for (int w = 0; w < kW; ++w) s4[w][e] = n4 + e < p.N ? p.w_scale[w][n4 + e] : 0.0f;
        b4[e] = biased && n4 + e < p.N ? p.bias[n4 + e] : 0.0f;
      }
    }
    cluster_wait();
    if (epi && !fail) {
      auto total4 = [&](int m, int w, float (&v)[4]) {
        const uint32_t at = red + (m * kW + w) * 512 + c4 * 4;
        uint4 x[kMaxSplit];
#pragma unroll
        for (int j = 0; j < kMaxSplit; ++j)
          if (j < p.split) x[j] = ld_cluster_v4(cluster_map(at, j));
        float4 t = make_float4(__uint_as_float(x[0].x), __uint_as_float(x[0].y),
                               __uint_as_float(x[0].z), __uint_as_float(x[0].w));
#pragma unroll
        for (int j = 1; j < kMaxSplit; ++j) {
          if (j < p.split) {
            t.x = add(t.x, __uint_as_float(x[j].x));
            t.y = add(t.y, __uint_as_float(x[j].y));
            t.z = add(t.z, __uint_as_float(x[j].z));
            t.w = add(t.w, __uint_as_float(x[j].w));
          }
        }
        v[0] = value(t.x);
        v[1] = value(t.y);
        v[2] = value(t.z);
        v[3] = value(t.w);
      };
#pragma unroll 1
      for (int m = first + (et >> 5); m < last; m += 8) {
        const float sa = lds_f32(sa_addr + m * 4);
        float v[4], g[4];
        total4(m, 0, v);
        if constexpr (kGated) total4(m, kW - 1, g);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v[e] = v[e] * sa * s4[0][e];
          if constexpr (kGated) v[e] = gated(v[e], g[e] * sa * s4[kW - 1][e], p.act);
          else if (biased) v[e] += b4[e];
        }
        const int64_t at = static_cast<int64_t>(m0 + m) * p.ldo + n4;
        if (p.rows16 && n4 + 4 <= p.N) {
          if (p.out_dtype == PK_F32)
            *reinterpret_cast<float4*>(static_cast<float*>(p.out) + at) =
                make_float4(v[0], v[1], v[2], v[3]);
          else
            *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + at) = make_uint2(
                pack16(p.out_dtype, v[0], v[1]), pack16(p.out_dtype, v[2], v[3]));
        } else {
          with_type(p.out, p.out_dtype, [&](auto* out) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (n4 + e < p.N) put(out + at + e, v[e]);
          });
        }
      }
    }
    // no CTA leaves while another fetches from its ring
    __syncwarp();
    cluster_arrive_unordered();
    cluster_wait();
    return;
  }

  tc_fence_before();
  if (__syncthreads_or(fail)) drain();
  if (warp == kMmaWarp) tmem_dealloc(tmem, p.tmem_cols);
}

// ---------------------------------------------------------------------------
// Many tokens: persistent CTA pairs, D[token, channel] tiles of 256 x 256
// (gated: 256 tokens x 128 outputs, gate and up side by side).
// ---------------------------------------------------------------------------
struct PairCfg {
  static constexpr int kATile = 128 * kBK;  // this CTA's 128 tokens
  static constexpr int kBTile = 128 * kBK;  // this CTA's 128 channels
  static constexpr int kStageBytes = kATile + kBTile;
  static constexpr int kStages = 6;
  static constexpr int kBarOff = kStages * kStageBytes;
  static constexpr int kScaleOff = kBarOff + 256;           // [2][256] scales, [2][256] bias
  static constexpr int kTurnOff = kScaleOff + 4 * 256 * 4;  // per epilogue warp [32][17] floats
  static constexpr int kTurnBytes = 32 * 17 * 4;
  static constexpr int kSmem = kTurnOff + kEpiWarps * kTurnBytes + 1024;
  static constexpr int kAccCols = 256;
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

constexpr int kGroupM = 8;

// Unit u of the schedule: tile (tm, tn), in how many parts, which part.
__device__ __forceinline__ void pair_unit(int u, const Params& p, int& tm, int& tn, int& parts,
                                          int& part) {
  int t = u;
  parts = 1;
  part = 0;
  if (u >= p.whole) {
    parts = p.parts;
    t = p.whole + (u - p.whole) / parts;
    part = (u - p.whole) % parts;
  }
  // rows of tiles in groups, so that the tiles in flight share operands in L2
  const int per_group = kGroupM * p.num_n;
  const int g = t / per_group;
  const int first = g * kGroupM;
  const int gm = min(p.num_m - first, kGroupM);
  tm = first + (t % per_group) % gm;
  tn = (t % per_group) / gm;
}

template <bool kE4M3, bool kGated>
__global__ void __launch_bounds__(kThreads, 1)
    w8a8_pair_kernel(const __grid_constant__ CUtensorMap tmA,
                     const __grid_constant__ CUtensorMap tmW0,
                     const __grid_constant__ CUtensorMap tmW1, const Params p) {
  using C = PairCfg;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  uint64_t* empty = full + C::kStages;
  uint64_t* acc_full = empty + C::kStages;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(acc_empty + 2);
  float* s_scale = reinterpret_cast<float*>(smem + C::kScaleOff);
  float* s_bias = s_scale + 2 * 256;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = static_cast<int>(cluster_ctarank());
  const int pair = blockIdx.x >> 1, npairs = gridDim.x >> 1;
  const int k_tiles = (p.K + kBK - 1) / kBK;
  const int num_units = p.whole + p.parts * (p.num_m * p.num_n - p.whole);
  constexpr int kTileN = kGated ? 128 : 256;  // outputs of a tile

  if (warp == kTmaWarp && lane == 0) {
    for (int i = 0; i < C::kStages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 2 * kEpiWarps);
    }
    fence_barrier_init();
    tma_prefetch_desc(&tmA);
    tma_prefetch_desc(&tmW0);
    if (kGated) tma_prefetch_desc(&tmW1);
  }
  if (warp == kMmaWarp) tmem_alloc_pair(tmem_holder, 512);
  tc_fence_before();
  cluster_sync();  // both CTAs' barriers exist before either signals the other
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  griddep_wait();
  griddep_launch_dependents();

  bool fail = false;
  if (warp == kTmaWarp) {
    const CUtensorMap* tmW = kGated && rank == 1 ? &tmW1 : &tmW0;
    const uint32_t full0 = cluster_map(smem_u32(&full[0]), 0);
    int st = 0;
    uint32_t parity = 1;
    for (int u = pair; u < num_units && !fail; u += npairs) {
      int tm, tn, parts, at;
      pair_unit(u, p, tm, tn, parts, at);
      const int row = tm * 256 + rank * 128;
      // this CTA's 128 / parts channels: of gate or up, or its half of the outputs
      const int boxes = 128 / parts / p.box;
      const int col = tn * kTileN + at * (kTileN / parts) + (kGated ? 0 : rank * (128 / parts));
      const uint32_t tx = 2u * (C::kATile + 128 / parts * kBK);
      for (int kt = 0; kt < k_tiles; ++kt) {
        fail = __any_sync(0xffffffffu, !mbar_wait(&empty[st], parity, p.status, kSiteW8PairProducer));
        if (fail) break;
        if (elect_one()) {
          uint8_t* base = smem + st * C::kStageBytes;
          const uint32_t bar = full0 + st * 8;
          if (rank == 0) mbar_arrive_expect_tx(&full[st], tx);
          tma_load_2d_pair(base, &tmA, bar, kt * kBK, row);
          for (int b = 0; b < boxes; ++b)
            tma_load_2d_pair(base + C::kATile + b * p.box * kBK, tmW, bar, kt * kBK, col + b * p.box);
        }
        __syncwarp();
        if (++st == C::kStages) {
          st = 0;
          parity ^= 1;
        }
      }
    }
  } else if (warp == kMmaWarp) {
    if (rank == 0) {
      const uint64_t desc0 = make_smem_desc(0, 16, 1024);
      const uint32_t base0 = smem_u32(smem);
      int local = 0, st = 0;
      uint32_t parity = 0;
      for (int u = pair; u < num_units && !fail; u += npairs, ++local) {
        const uint32_t idesc = idesc8(kE4M3, 256, u < p.whole ? 256 : 256 / p.parts);
        const int ab = local & 1;
        if (local >= 2)
          fail = __any_sync(0xffffffffu, !mbar_wait_cluster(&acc_empty[ab], ((local >> 1) - 1) & 1,
                                                            p.status, kSiteW8PairMma));
        if (fail) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem + ab * C::kAccCols;
        for (int kt = 0; kt < k_tiles; ++kt) {
          fail = __any_sync(0xffffffffu, !mbar_wait(&full[st], parity, p.status, kSiteW8PairMma));
          if (fail) break;
          if (elect_one()) {
            const uint64_t ad = desc0 + ((base0 + st * C::kStageBytes) >> 4);
            const uint64_t bd = ad + (C::kATile >> 4);
#pragma unroll
            for (int s = 0; s < kKSteps; ++s)
              umma8_pair<kE4M3>(d_tmem, ad + (s * 32 >> 4), bd + (s * 32 >> 4), idesc,
                                (kt > 0 || s > 0) ? 1u : 0u);
            umma_commit_pair(&empty[st]);
            if (kt + 1 == k_tiles) umma_commit_pair(&acc_full[ab]);
          }
          __syncwarp();
          if (++st == C::kStages) {
            st = 0;
            parity ^= 1;
          }
        }
      }
    }
  } else {
    // ---- epilogue (both CTAs): a thread holds one token's row ----
    const int q = warp & 3;  // TMEM lane quarter this warp may access
    const int part = (warp - kEpiWarp0) >> 2;  // which of two 32-output runs
    const int et = tid - kEpiWarp0 * 32;
    const uint32_t acc_empty0 = cluster_map(smem_u32(&acc_empty[0]), 0);
    int local = 0;
    for (int u = pair; u < num_units && !fail; u += npairs, ++local) {
      int tm, tn, parts, at;
      pair_unit(u, p, tm, tn, parts, at);
      const int ab = local & 1;
      const int outs = kTileN / parts;  // outputs of this unit
      const int n0 = tn * kTileN + at * outs;
      // this unit's channel scales (gate then up) and bias
      float* sc = s_scale + ab * 256;
      float* bs = s_bias + ab * 256;
      const uint32_t sc_addr = smem_u32(sc);
      constexpr int kBiasOff = 2 * 256 * 4;  // from a unit's scales to its bias
      for (int i = et; i < (kGated ? 2 * outs : outs); i += kEpiThreads) {
        const int w = kGated && i >= outs ? 1 : 0;
        const int n = n0 + i - w * outs;
        sc[i] = n < p.N ? p.w_scale[w][n] : 0.0f;
        if (!kGated) bs[i] = p.bias != nullptr && n < p.N ? p.bias[n] : 0.0f;
      }
      const int row = tm * 256 + rank * 128 + q * 32 + lane;
      const float sa = row < p.M ? p.a_scale[row] : 0.0f;
      // one barrier a unit: the scales are in place, and the warps agree on
      // whether the wait ran out (none is left waiting for one that gave up)
      fail = named_bar_or(
          1, kEpiThreads,
          !mbar_wait(&acc_full[ab], (local >> 1) & 1, p.status, kSiteW8PairEpilogue));
      if (fail) break;
      tc_fence_after();
      const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16) + ab * C::kAccCols;
#pragma unroll 1
      for (int c = part * 32; c < outs; c += 64) {
        uint32_t x[32], y[32];
        tmem_ld_32x32b_x32(taddr + c, x);
        if (kGated) tmem_ld_32x32b_x32(taddr + outs + c, y);
        tmem_ld_wait();
        // all values before the first store: it would hold back later reads
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          float w[4];
          lds_floats(sc_addr + (c + i) * 4, w);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[i + e] = acc_value<kE4M3>(x[i + e]) * sa * w[e];
          if constexpr (kGated) {
            lds_floats(sc_addr + (outs + c + i) * 4, w);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              v[i + e] = gated(v[i + e], acc_value<kE4M3>(y[i + e]) * sa * w[e], p.act);
          } else if (p.bias != nullptr) {
            lds_floats(sc_addr + kBiasOff + (c + i) * 4, w);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[i + e] += w[e];
          }
        }
        const uint32_t turn = smem_u32(smem + C::kTurnOff) + (warp - kEpiWarp0) * C::kTurnBytes;
        const int64_t row0 = static_cast<int64_t>(row) - lane;
        if (p.rows16) {
          // 64 bytes of each of the warp's rows through shared memory (the
          // 16-byte pieces of a row pair rotated so that neither side has bank
          // conflicts), so that a store covers eight rows' whole sectors: stored
          // by the row's own thread a tile's epilogue took 5 us.
          const int elt = p.out_dtype == PK_F32 ? 4 : 2;
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            if (g == 1 && elt == 2) break;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const uint32_t at = turn + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4);
              if (elt == 4)
                sts_v4f(at, v[16 * g + 4 * j], v[16 * g + 4 * j + 1], v[16 * g + 4 * j + 2],
                        v[16 * g + 4 * j + 3]);
              else
                sts_v4u(at, pack16(p.out_dtype, v[8 * j], v[8 * j + 1]),
                        pack16(p.out_dtype, v[8 * j + 2], v[8 * j + 3]),
                        pack16(p.out_dtype, v[8 * j + 4], v[8 * j + 5]),
                        pack16(p.out_dtype, v[8 * j + 6], v[8 * j + 7]));
            }
            __syncwarp();
            const int j = lane & 3, per = 16 / elt;  // this lane's piece of a row, its outputs
            const int n = n0 + c + 16 * g + j * per;
#pragma unroll
            for (int r = 0; r < 32; r += 8) {
              const int rr = r + (lane >> 2);
              const uint4 w = lds_v4(turn + rr * 64 + ((j ^ ((rr >> 1) & 3)) << 4));
              if (n < p.N && row0 + rr < p.M) {
                uint8_t* o = static_cast<uint8_t*>(p.out) + ((row0 + rr) * p.ldo + n) * elt;
                if (n + per <= p.N) {
                  *reinterpret_cast<uint4*>(o) = w;
                } else {
                  const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                  for (int k = 0; k < 4; ++k) {
                    if (elt == 4) {
                      if (n + k < p.N) reinterpret_cast<uint32_t*>(o)[k] = words[k];
                    } else {
                      if (n + 2 * k < p.N) reinterpret_cast<uint16_t*>(o)[2 * k] = static_cast<uint16_t>(words[k]);
                      if (n + 2 * k + 1 < p.N) reinterpret_cast<uint16_t*>(o)[2 * k + 1] = static_cast<uint16_t>(words[k] >> 16);
                    }
                  }
                }
              }
            }
            __syncwarp();
          }
        } else {
          // Rows off 16-byte boundaries: sixteen columns at a time through
          // shared memory, so that a warp stores two rows' runs at once (333 x
          // 1111 x 1001: 16 us, with single stores of 32 rows 52).
#pragma unroll
          for (int g = 0; g < 32; g += 16) {
#pragma unroll
            for (int i = 0; i < 16; ++i) sts_f32(turn + (lane * 17 + i) * 4, v[g + i]);
            __syncwarp();
            const int n = n0 + c + g + (lane & 15);
            with_type(p.out, p.out_dtype, [&](auto* out) {
#pragma unroll
              for (int r = 0; r < 32; r += 2) {
                const int64_t at = row0 + r + (lane >> 4);
                const float f = lds_f32(turn + ((r + (lane >> 4)) * 17 + (lane & 15)) * 4);
                if (n < p.N && at < p.M) put(out + at * p.ldo + n, f);
              }
            });
            __syncwarp();
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(acc_empty0 + ab * 8);
    }
  }

  tc_fence_before();
  if (__syncthreads_or(fail)) drain();
  cluster_sync();  // neither CTA leaves while the other may still touch its memory
  tc_fence_after();
  if (warp == kMmaWarp) tmem_dealloc_pair(tmem, 512);
}

// ---------------------------------------------------------------------------
// launch
// ---------------------------------------------------------------------------
int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

bool rows_map(CUtensorMap* m, const void* base, int64_t rows, int64_t K, int64_t ld, int box_rows,
              const char** why) {
  return encode_tmap_2d(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, K, rows, ld, kBK, box_rows,
                        CU_TENSOR_MAP_SWIZZLE_128B, why);
}

Params params_of(const W8A8Args& g) {
  Params p{};
  p.a_scale = g.a_scale;
  p.w_scale[0] = g.w_scale[0];
  p.w_scale[1] = g.w_scale[1];
  p.bias = g.bias;
  p.out = g.out;
  p.ldo = g.ldo;
  p.M = static_cast<int>(g.M);
  p.N = static_cast<int>(g.N);
  p.K = static_cast<int>(g.K);
  p.out_dtype = g.out_dtype;
  p.act = g.act;
  p.rows16 = (reinterpret_cast<uintptr_t>(g.out) & 15) == 0 &&
             (g.ldo * (g.out_dtype == PK_F32 ? 4 : 2)) % 16 == 0;
  p.split = 1;
  p.status = g.status;
  return p;
}

constexpr int kMaxSmem = 226 * 1024;  // for a ring and what follows it
constexpr int kAllSmem = 227 * 1024;

template <typename Kernel>
cudaError_t launch(Kernel kernel, int grid, int threads, int cluster, int smem, cudaStream_t s,
                   const CUtensorMap (&tm)[3], const Params& p) {
  // the attribute once and for all sizes (a plan's size changes from call to call)
  cudaError_t e = set_max_smem(reinterpret_cast<const void*>(kernel), kAllSmem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attrs[2];
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = cluster;
  attrs[1].val.clusterDim.y = 1;
  attrs[1].val.clusterDim.z = 1;
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = attrs;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kernel, tm[0], tm[1], tm[2], p);
}

// Which kernel, how many tokens a tile, how many K splits: from the sizes alone.
struct Plan {
  bool pair;
  int nt, split;
  bool deep;   // swap: the ring may take a whole SM's shared memory
  int pieces;  // swap: accumulators of a CTA
};

// Shared memory of a swap CTA: its ring, and what follows it.
struct SwapSmem {
  int stages, stage_bytes, own_red, bytes, tmem_cols;
  bool fits;
};

SwapSmem swap_smem(const Plan& plan, bool gated, int64_t k_tiles) {
  SwapSmem c{};
  const int w = gated ? 2 : 1;
  const int sums = plan.split > 1 ? w * plan.nt * 128 * 4 : 0;
  c.stage_bytes = w * kWTile + plan.nt * kBK;
  c.own_red = sums > 0 && sums <= 16 * 1024;
  const int rest = kMaxTokens * 4 + kSwapBars + (c.own_red ? sums : 0) + 1024;
  // two CTAs an SM where half the memory holds four stages
  const int half = kMaxSmem / 2 - rest, whole = kMaxSmem - rest;
  c.stages = (!plan.deep && half / c.stage_bytes >= 4 ? half : whole) / c.stage_bytes;
  c.stages = static_cast<int>(std::min<int64_t>(std::min(c.stages, 12), ceil_div(k_tiles, plan.split)));
  // sums without memory of their own go into the drained ring
  if (sums > 0 && !c.own_red)
    while (c.stages * c.stage_bytes < sums && (c.stages + 1) * c.stage_bytes <= whole) ++c.stages;
  c.fits = sums == 0 || c.own_red || sums <= c.stages * c.stage_bytes;
  c.bytes = c.stages * c.stage_bytes + rest;
  c.tmem_cols = 32;
  while (c.tmem_cols < plan.nt * w * plan.pieces) c.tmem_cols *= 2;
  return c;
}

template <bool kE4M3, bool kGated>
cudaError_t launch_swap(const W8A8Args& g, const Plan& plan, cudaStream_t s, const char** why) {
  const SwapSmem c = swap_smem(plan, kGated, ceil_div(g.K, kBK));
  if (!c.fits) {
    *why = "the sums of the K split do not fit shared memory";
    return cudaErrorInvalidValue;
  }
  CUtensorMap tm[3];
  if (!rows_map(&tm[0], g.a, g.M, g.K, g.lda, plan.nt, why) ||
      !rows_map(&tm[1], g.w[0], g.N, g.K, g.ldw[0], 128, why))
    return cudaErrorInvalidValue;
  tm[2] = tm[1];
  if (kGated && !rows_map(&tm[2], g.w[1], g.N, g.K, g.ldw[1], 128, why))
    return cudaErrorInvalidValue;
  Params p = params_of(g);
  p.nt = plan.nt;
  p.split = plan.split;
  p.stages = c.stages;
  p.stage_bytes = c.stage_bytes;
  p.own_red = c.own_red;
  p.pieces = plan.pieces;
  p.tmem_cols = c.tmem_cols;
  p.num_m = static_cast<int>(ceil_div(g.M, plan.nt));
  p.num_n = static_cast<int>(ceil_div(g.N, 128));
  const int64_t grid = static_cast<int64_t>(p.num_m) * p.num_n * p.split;
  if (grid >= (1ll << 31)) return cudaErrorInvalidConfiguration;
  return launch(w8a8_swap_kernel<kE4M3, kGated>, static_cast<int>(grid), kThreads, p.split, c.bytes,
                s, tm, p);
}

// A partial wave (the last, or all there is) runs as narrower units, two or four
// a tile, where they still fit one wave: a half unit takes 0.75 of a tile's
// time, a quarter 0.55.
void pair_schedule(int64_t tiles, int slots, int* whole, int* parts) {
  const int64_t tail = tiles % slots;
  *parts = tail == 0 ? 1 : 4 * tail <= slots ? 4 : 2 * tail <= slots ? 2 : 1;
  *whole = static_cast<int>(*parts == 1 ? tiles : tiles - tail);
}

template <bool kE4M3, bool kGated>
cudaError_t launch_pair(const W8A8Args& g, cudaStream_t s, const char** why) {
  Params p = params_of(g);
  p.num_m = static_cast<int>(ceil_div(g.M, 256));
  p.num_n = static_cast<int>(ceil_div(g.N, kGated ? 128 : 256));
  if (static_cast<int64_t>(p.num_m) * p.num_n >= 1 << 29) return cudaErrorInvalidConfiguration;
  const int tiles = p.num_m * p.num_n;
  const int slots = num_sms() / 2;
  pair_schedule(tiles, slots, &p.whole, &p.parts);
  p.box = p.parts == 4 ? 32 : 64;
  CUtensorMap tm[3];
  if (!rows_map(&tm[0], g.a, g.M, g.K, g.lda, 128, why) ||
      !rows_map(&tm[1], g.w[0], g.N, g.K, g.ldw[0], p.box, why))
    return cudaErrorInvalidValue;
  tm[2] = tm[1];
  if (kGated && !rows_map(&tm[2], g.w[1], g.N, g.K, g.ldw[1], p.box, why))
    return cudaErrorInvalidValue;
  const int units = p.whole + p.parts * (tiles - p.whole);
  return launch(w8a8_pair_kernel<kE4M3, kGated>, 2 * (units < slots ? units : slots),
                kThreads, 2, PairCfg::kSmem, s, tm, p);
}

// Estimated microseconds of a plan, from the kernels' measured parts (what
// matters is the order of the plans):
//  * an SM takes in ~150 GB/s of tiles, and no more than its rings hold per
//    ~1.6 us of memory latency; HBM delivers ~6.3 TB/s of weights
//    to all SMs, less to a part of them;
//  * a CTA spends 0.1 us on a K tile's barriers and 30 ns on an MMA, or, from 114
//    tokens on, the MMA's own nt / 2 cycles;
//  * a grid runs in rounds of the CTAs that are resident at once: at one CTA an
//    SM 148, of clusters of 4 132, of clusters of 8 120;
//  * swap: 2.5 us of launch and first loads, 0.7 more where a CTA takes most of an
//    SM's memory (the next kernel's CTAs then wait for it); per token of a tile
//    13 ns of epilogue (gated 23), with a K split 0.8 us + nt * (5 + 40 / split) ns a
//    weight;
//  * pair: 6 us around the main loop, 0.28 us a K tile (0.21 of a half unit, 0.155
//    of a quarter).
constexpr float kSmBytes = 150e3f, kHbmBytes = 6.3e6f, kLatency = 1.6f;  // per us; us

float plan_us(const Plan& plan, const W8A8Args& g) {
  const float sms = static_cast<float>(num_sms());
  const float w = g.gated ? 2.0f : 1.0f;
  const int64_t k_tiles = ceil_div(g.K, kBK);
  if (plan.pair) {
    const int64_t num_m = ceil_div(g.M, 256), tiles = num_m * ceil_div(g.N, g.gated ? 128 : 256);
    const int slots = num_sms() / 2;
    int whole, parts;
    pair_schedule(tiles, slots, &whole, &parts);
    const float kt = static_cast<float>(k_tiles), weights = 256.0f * kBK / static_cast<float>(num_m);
    auto wave = [&](int64_t units, float k_tile_us) {
      return kt * std::max(static_cast<float>(units) * weights / kHbmBytes, k_tile_us);
    };
    float us = 6.0f + static_cast<float>(whole / slots) * wave(slots, 0.28f);
    if (tiles % slots > 0)
      us += wave(tiles % slots, parts == 4 ? 0.155f : parts == 2 ? 0.21f : 0.28f);
    return us;
  }
  const SwapSmem c = swap_smem(plan, g.gated, k_tiles);
  const int occ = c.bytes <= kMaxSmem / 2 ? 2 : 1;
  const int64_t num_m = ceil_div(g.M, plan.nt);
  const int64_t ctas = num_m * ceil_div(g.N, 128) * plan.split;
  const float part = plan.split == 8 ? 120.0f / 148 : plan.split == 4 ? 132.0f / 148 : 1.0f;
  const int64_t one = std::max<int64_t>(1, static_cast<int64_t>(sms * part));  // CTAs at one an SM
  const float kt = static_cast<float>(ceil_div(k_tiles, plan.split));
  const float ring = static_cast<float>(c.stages * c.stage_bytes);
  const float nt = static_cast<float>(plan.nt), split = static_cast<float>(plan.split);
  const float stage = static_cast<float>(c.stage_bytes), mma = std::max(0.030f, nt / 2 / 1900);
  auto round = [&](int64_t n) {  // us of n resident CTAs, up to their epilogues
    const float per_sm = static_cast<float>(ceil_div(n, one));
    const float busy = std::min(1.0f, static_cast<float>(n) / sms);
    const float hbm = static_cast<float>(n) * w * kWTile / static_cast<float>(num_m) /
                      (kHbmBytes * (0.3f + 0.7f * busy));
    const float in = std::max(per_sm * stage / kSmBytes, stage * kLatency / ring);
    const float issue = std::max(0.1f + 4 * w * mma, per_sm * 4 * w * mma);
    return kt * std::max({hbm, in, issue});
  };
  const float epilogue = plan.split == 1
                             ? nt * (g.gated ? 0.023f : 0.013f)
                             : 0.8f + w * nt * (0.005f + 0.040f / split);
  // two CTAs on an SM: a fifth of an epilogue hides behind the other's
  const int64_t full = ctas / (one * occ), rest = ctas % (one * occ);
  float us = (c.bytes > kMaxSmem / 2 ? 3.2f : 2.5f) +
             static_cast<float>(full) * (round(one * occ) + epilogue * (occ == 2 ? 1.8f : 1.0f));
  if (rest > 0) us += round(rest) + epilogue * (rest > one ? 1.8f : 1.0f);
  return us;
}

// An e4m3 MMA loses a part of its accumulator's last place at each step, always
// towards zero: measured 4.5e-9 of the result a step of 32, 1e-6 after 7168 of
// K. So an accumulator takes a limited number of K tiles, and the K splits and
// pieces of a swap CTA are added up in fp32: 40 tiles (7e-7) where the output is fp32,
// 1280 (2.3e-5, a twentieth of fp16's half step) where it has 16 bits. A tile of 16
// tokens holds 32 accumulators a CTA (gated 16) in a split of 8: fp32 outputs of more
// than 1310720 of K (gated 655360) have longer pieces, evenly. The pair kernel has one
// accumulator.
constexpr int kPieceF32 = 40, kPiece16 = 1280;

Plan search(const W8A8Args& g) {
  const int64_t k_tiles = ceil_div(g.K, kBK);
  const int64_t limit = !g.e4m3 ? k_tiles : g.out_dtype == PK_F32 ? kPieceF32 : kPiece16;
  Plan best{true, 0, 1, false, 1};
  float least = g.M > 128 && k_tiles <= limit ? plan_us(best, g) : 1e30f;
  int64_t fewest = 1ll << 60;  // K tiles over the limit in an accumulator, 0 before all else
  if (least < 1e30f) fewest = 0;
  auto consider = [&](int nt) {
    for (int split = 1; split <= kMaxSplit && split <= k_tiles; split *= 2) {
      for (int deep = 0; deep < 2; ++deep) {
        Plan plan{false, nt, split, deep != 0, 1};
        if (!swap_smem(plan, g.gated, k_tiles).fits) continue;
        const int64_t kt = ceil_div(k_tiles, split);
        const int cols = plan.nt * (g.gated ? 2 : 1);
        while (plan.pieces * limit < kt && 2 * plan.pieces * cols <= (deep ? 512 : 256)) plan.pieces *= 2;
        const int64_t over = std::max<int64_t>(0, ceil_div(kt, plan.pieces) - limit);
        const float us = plan_us(plan, g);
        if (over < fewest || (over == fewest && us < least)) {
          fewest = over;
          least = us;
          best = plan;
        }
      }
    }
  };
  // token tiles as even as sixteens allow, from as few as there can be to 16 wide
  int last = 0;
  for (int64_t num_m = ceil_div(g.M, kMaxTokens); num_m <= ceil_div(g.M, 256) + 16 && last != 16;
       ++num_m) {
    const int nt = static_cast<int>(ceil_div(ceil_div(g.M, num_m), 16) * 16);
    if (nt != last) consider(nt);
    last = nt;
  }
  // the narrower, the more accumulators
  while (fewest > 0 && last > 16) consider(last -= 16);
  return best;
}

// The plans of recent sizes, per host thread (a decode loop asks for the same
// few; a search is several microseconds): a function of the sizes alone.
Plan plan_of(const W8A8Args& g) {
  struct Entry {
    int64_t M, N, K;
    int key, sms;
    Plan plan;
  };
  static thread_local Entry cache[64] = {};
  const int key = 1 + (g.gated ? 2 : 0) + (g.e4m3 ? 4 : 0) + (g.out_dtype == PK_F32 ? 8 : 0);
  const uint64_t hash = (static_cast<uint64_t>(g.M) * 0x9E3779B97F4A7C15ull ^
                         static_cast<uint64_t>(g.N) * 0xC2B2AE3D27D4EB4Full ^
                         static_cast<uint64_t>(g.K) * 0x165667B19E3779F9ull) + key;
  Entry& e = cache[(hash ^ hash >> 32 ^ hash >> 17) & 63];
  const int sms = num_sms();
  if (e.M != g.M || e.N != g.N || e.K != g.K || e.key != key || e.sms != sms)
    e = Entry{g.M, g.N, g.K, key, sms, search(g)};
  return e.plan;
}

template <bool kE4M3, bool kGated>
cudaError_t launch_typed(const W8A8Args& g, cudaStream_t s, const char** why) {
  const Plan plan = plan_of(g);
  return plan.pair ? launch_pair<kE4M3, kGated>(g, s, why) : launch_swap<kE4M3, kGated>(g, plan, s, why);
}

}  // namespace

cudaError_t launch_w8a8(const W8A8Args& g, cudaStream_t s, const char** why) {
  if (g.gated)
    return g.e4m3 ? launch_typed<true, true>(g, s, why) : launch_typed<false, true>(g, s, why);
  return g.e4m3 ? launch_typed<true, false>(g, s, why) : launch_typed<false, false>(g, s, why);
}

}  // namespace pk
