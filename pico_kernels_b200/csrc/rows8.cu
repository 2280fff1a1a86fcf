// Rows in 8 bits: the quantizer of activations and weights with one scale per
// row, its inverse, and the RMS norm that writes its output already quantized.
//
//   quantize      a = max(max_k |x_k|, 1e-12),  scale = a / most,
//                 q_k = round(x_k * most / a),  most = 127 (int8) or 448 (e4m3)
//   rms norm      h = T(x + residual),  r = 1 / sqrt(mean(h^2) + eps),
//                 y_k = h_k * r * w_k, quantized as above
//   dequantize    x_k = q_k * scale
//
// All three are bound by HBM: a row is read once, kept while its sum and its
// largest magnitude are reduced, and written once (4096 x 28672 bf16 to e4m3
// 54 us = 6.5 TB/s; the norm of 4096 x 8192 with a residual 40 us = 5.9 TB/s,
// without one 23.6 us = 4.3 TB/s, where about 16 instructions a value and the
// reduction's round trip between a row's passes take longer than its bytes).
// The norm needs one reduction, not two (the sum for r, then the maximum of y): r multiplies
// the whole row, so the codes of y are those of u_k = h_k * w_k, and the sum of
// h^2 and the maximum of |u| are reduced together; r enters the scale alone.
// The maximum propagates NaN (across threads on the bit patterns of |u|, ordered
// like the values with infinities and NaN on top), so none can be lost in it.
//
// A row that holds a NaN or an infinity has no 8-bit form: it gets scale NaN
// and codes 0, so that every product with it is NaN and no other row is
// touched. Sums, maxima and scales are fp32; the only roundings to fewer bits
// are the stored h (the residual stream's own type, which is what the next
// layer adds to, so the norm is that of the stored value) and the codes, which are
// the nearest to quotients that carry one fp32 rounding: a half step is met as
// such, and goes to even.
#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

#include "pk_common.cuh"

namespace pk {
namespace {

constexpr float kTiny = 1e-12f;     // smallest row maximum, as in the int4 group scales
constexpr uint32_t kInfBits = 0x7f800000u;
constexpr int kMaxLanes = 512;      // threads of a row
constexpr int kMostStaged = 225 * 1024;  // shared memory for rows in flight

struct RowsParams {
  const void* x;
  const void* residual;  // norm: added to x (nullptr: none)
  const void* weight;    // norm: fp32, or x's type
  void* h;               // norm with a residual: the sum, in x's type
  uint8_t* q;
  float* scale;
  int64_t ldx, ldr, ldh, ldq;
  uint32_t sx, sr, sh, sq;  // the same in bytes
  int64_t rows;
  int cols;
  int lanes;             // threads of a row
  int stages;            // rows in flight per group of threads
  int slot;              // bytes of one staged row
  int weight_f32;
  int codes_vec;         // rows of codes 8-byte aligned
  int e4m3;
  float eps;
  float inv_cols;
};

template <typename T>
__device__ __forceinline__ float as_f32(T v);
template <>
__device__ __forceinline__ float as_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float as_f32<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float as_f32<float>(float v) { return v; }

template <typename T>
__device__ __forceinline__ T as_type(float v);
template <>
__device__ __forceinline__ __half as_type<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 as_type<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ float as_type<float>(float v) { return v; }

// Eight consecutive values as they lie in memory: two of a 16-bit type stay in
// one register until they are used (arrays of T made the compiler spread them
// over eight, and a row of several chunks spilled).
template <typename T>
struct Eight {
  static constexpr int kWords = sizeof(T) * 2;
  uint32_t w[kWords];

  __device__ __forceinline__ void values(float (&v)[8]) const {
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(w[j]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        v[2 * j] = f.x;
        v[2 * j + 1] = f.y;
      }
    }
  }

  __device__ __forceinline__ void round(const float (&v)[8]) {
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(v[j]);
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&p);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const __half2 p = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&p);
      }
    }
  }

  __device__ __forceinline__ T element(int j) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[j]);
    } else {
      const uint16_t h = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
      return *reinterpret_cast<const T*>(&h);
    }
  }
};

// 16 bytes of a row (from L2: read once, and perhaps just written) or of the
// norm's weights (kept in L1: every row of the SM reads them; not as read-only
// data, since the kernel before this one may still write them when it starts).
template <bool kWeights>
__device__ __forceinline__ uint4 load16(const uint4* p) {
  return kWeights ? __ldca(p) : __ldcg(p);
}

// 16-byte accesses (two for fp32).
template <typename T, bool kWeights>
__device__ __forceinline__ Eight<T> load8(const T* p) {
  Eight<T> e;
#pragma unroll
  for (int i = 0; i < Eight<T>::kWords / 4; ++i) {
    const uint4 v = load16<kWeights>(reinterpret_cast<const uint4*>(p) + i);
    e.w[4 * i] = v.x;
    e.w[4 * i + 1] = v.y;
    e.w[4 * i + 2] = v.z;
    e.w[4 * i + 3] = v.w;
  }
  return e;
}

template <int kWords, int kSkip>
__device__ __forceinline__ void shift_words(const uint32_t (&in)[kWords + 4], int bits,
                                            uint32_t (&out)[kWords]) {
#pragma unroll
  for (int i = 0; i < kWords; ++i) out[i] = __funnelshift_r(in[i + kSkip], in[i + kSkip + 1], bits);
}

// kWords words from byte `off` of in[].
template <int kWords>
__device__ __forceinline__ void shift_any(const uint32_t (&in)[kWords + 4], int off,
                                          uint32_t (&out)[kWords]) {
  const int bits = (off & 3) * 8;
  switch (off >> 2) {
    case 0: shift_words<kWords, 0>(in, bits, out); break;
    case 1: shift_words<kWords, 1>(in, bits, out); break;
    case 2: shift_words<kWords, 2>(in, bits, out); break;
    default: shift_words<kWords, 3>(in, bits, out); break;
  }
}

// load8 from an address that is aligned to its element only: the aligned
// 16-byte blocks that hold the values (each holds at least one of them), and
// a shift by the distance, which is the same for all chunks of a row.
template <typename T, bool kWeights>
__device__ __forceinline__ Eight<T> load8_shifted(const T* p) {
  constexpr int kWords = Eight<T>::kWords;
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 15);
  const uint4* base = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p) - off);
  uint32_t in[kWords + 4];
#pragma unroll
  for (int i = 0; i < kWords / 4 + 1; ++i) {
    const uint4 v =
        i < kWords / 4 || off != 0 ? load16<kWeights>(base + i) : make_uint4(0, 0, 0, 0);
    in[4 * i] = v.x;
    in[4 * i + 1] = v.y;
    in[4 * i + 2] = v.z;
    in[4 * i + 3] = v.w;
  }
  Eight<T> e;
  shift_any<kWords>(in, off, e.w);
  return e;
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const Eight<T>& e) {
#pragma unroll
  for (int i = 0; i < Eight<T>::kWords / 4; ++i)
    reinterpret_cast<uint4*>(p)[i] =
        make_uint4(e.w[4 * i], e.w[4 * i + 1], e.w[4 * i + 2], e.w[4 * i + 3]);
}

// Columns c0 .. c0 + 7 of a row of `cols`, 0 past its end.
template <typename T, bool kWeights = false>
__device__ __forceinline__ Eight<T> load_row8(const T* row, int c0, int cols) {
  if (c0 + 8 <= cols)
    return (reinterpret_cast<uintptr_t>(row + c0) & 15) == 0 ? load8<T, kWeights>(row + c0)
                                                             : load8_shifted<T, kWeights>(row + c0);
  Eight<T> e;
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = c0 + j < cols ? as_f32<T>(row[c0 + j]) : 0.0f;
  e.round(v);  // the values themselves
  return e;
}

// Columns c0 .. c0 + 7 of the norm's weights; kWhole: aligned and whole.
template <typename W, bool kWhole>
__device__ __forceinline__ Eight<W> load_weights(const W* w, int c0, int cols) {
  if constexpr (kWhole) return load8<W, true>(w + c0);
  else return load_row8<W, true>(w, c0, cols);
}

// e + r, rounded to the stream's type. Two 16-bit values at a time: the sum of
// two such numbers is rounded once (the same bits as an fp32 addition and a
// rounding: fp32 holds every sum in which both matter), in one instruction
// where unpacking, adding and packing took seven.
template <typename T>
__device__ __forceinline__ void add(Eight<T>& e, const Eight<T>& r) {
#pragma unroll
  for (int i = 0; i < Eight<T>::kWords; ++i) {
    if constexpr (std::is_same<T, float>::value) {
      e.w[i] = __float_as_uint(__uint_as_float(e.w[i]) + __uint_as_float(r.w[i]));
    } else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      asm("add.rn.bf16x2 %0, %1, %2;" : "=r"(e.w[i]) : "r"(e.w[i]), "r"(r.w[i]));
    } else {
      asm("add.rn.f16x2 %0, %1, %2;" : "=r"(e.w[i]) : "r"(e.w[i]), "r"(r.w[i]));
    }
  }
}

template <typename T>
__device__ __forceinline__ void store_row8(T* row, int c0, int cols, const Eight<T>& e) {
  if (c0 + 8 <= cols && (reinterpret_cast<uintptr_t>(row + c0) & 15) == 0) {
    store8<T>(row + c0, e);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c0 + j < cols) row[c0 + j] = e.element(j);
  }
}

// store_row8 by a whole warp to rows that start off a 16-byte boundary, every
// lane the chunk after its neighbour's (`first`, `last`: a lane without a
// neighbour below or above it in the row): the 16-byte blocks that hold the end
// of its own chunk and the start of the next lane's, and single values only
// where no block is. Norm with a residual, 5000 x 5001 bf16: 63 us (60 when the two
// were compared), by single
// values 86; in fp32 single values are faster (3000 x 1001: 21.7 us, so 28.2).
template <typename T>
__device__ __forceinline__ void store_shifted8(T* row, int c0, int cols, const Eight<T>& e,
                                               bool first, bool last) {
  constexpr int kWords = Eight<T>::kWords;
  uint32_t in[kWords + 4];
#pragma unroll
  for (int i = 0; i < kWords; ++i) in[i] = e.w[i];
#pragma unroll
  for (int i = 0; i < 4; ++i) in[kWords + i] = __shfl_down_sync(0xffffffffu, e.w[i], 1);
  // bytes and values of a chunk before its first boundary, the same for the row
  const int before = static_cast<int>(-reinterpret_cast<uintptr_t>(row) & 15);
  const int head = before / static_cast<int>(sizeof(T));
  Eight<T> s;
  shift_any<kWords>(in, before, s.w);
  const bool block = (head == 0 || !last) && c0 + head + 8 <= cols;
  const bool start = head == 0 || (!first && c0 + head <= cols);  // [0, head) is in a block
  if (block) store8<T>(row + c0 + head, s);
  if (!block || !start) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c0 + j < cols && !(j < head ? start : block)) row[c0 + j] = e.element(j);
  }
}

// What takes a row's u to its codes: most / max|u| as the sum of two fp32 numbers
// (both 0: the row has no 8-bit form).
struct Factor {
  float hi, lo;
};

__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}

// Two quotients u * most / max|u|, each rounded to fp32 once (off by 2^-24 of
// itself): with the factor as one fp32 number a quotient that is a half step of
// the codes came out beside it, and values of 16 bits hit half steps often. It
// costs a packed multiplication per two values, and int8 a packed addition (codes
// 4096 x 11008 22.1 -> 23.8 us; the norm of 4096 x 8192 22.5 -> 23.6, with a residual
// nothing).
__device__ __forceinline__ uint64_t quotients2(float a, float b, Factor f) {
  const uint64_t u = pack2(a, b);
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(u), "l"(pack2(f.lo, f.lo)));
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(r) : "l"(u), "l"(pack2(f.hi, f.hi)));
  return r;
}

// Four int8 codes: adding 1.5 * 2^23 leaves the quotient, rounded half to even by
// the addition, as an integer in the low bits. A quotient is at most 127 and a
// last place, so no code passes 127.
__device__ __forceinline__ uint32_t int8_codes4(const float* u, Factor f) {
  constexpr float kMagic = 12582912.0f;
  uint64_t a = quotients2(u[0], u[1], f), b = quotients2(u[2], u[3], f);
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(a) : "l"(pack2(kMagic, kMagic)));
  asm("add.rn.f32x2 %0, %0, %1;" : "+l"(b) : "l"(pack2(kMagic, kMagic)));
  return prmt(prmt(static_cast<uint32_t>(a), static_cast<uint32_t>(a >> 32), 0x0040),
              prmt(static_cast<uint32_t>(b), static_cast<uint32_t>(b >> 32), 0x0040), 0x5410);
}

// Largest of |a|, |b|, |c|; NaN if one is NaN.
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(fabsf(b)), "f"(fabsf(c)));
  return r;
}

// Largest |value| of both halves of two words of a 16-bit type, NaN if one is; the
// signs of the result mean nothing.
template <typename T>
__device__ __forceinline__ uint32_t max2_abs(uint32_t a, uint32_t b) {
  uint32_t r;
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  else
    asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

template <bool kE4M3>
__device__ __forceinline__ uint32_t codes4(const float* u, Factor f) {
  if constexpr (kE4M3) {
    const uint32_t lo =
        __nv_cvt_float2_to_fp8x2(unpack2(quotients2(u[0], u[1], f)), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi =
        __nv_cvt_float2_to_fp8x2(unpack2(quotients2(u[2], u[3], f)), __NV_SATFINITE, __NV_E4M3);
    return prmt(lo, hi, 0x5410);
  } else {
    return int8_codes4(u, f);
  }
}

// Codes of the chunk at column c0: whole where every chunk of the matrix is
// (kWhole), else as the row's end and the caller's pitch allow.
template <bool kE4M3, bool kWhole>
__device__ __forceinline__ void store_codes(uint8_t* q, int c0, int cols, bool vec,
                                            const float (&u)[8], Factor f) {
  const uint32_t lo = codes4<kE4M3>(u, f), hi = codes4<kE4M3>(u + 4, f);
  if (kWhole || (vec && c0 + 8 <= cols)) {
    *reinterpret_cast<uint2*>(q + c0) = make_uint2(lo, hi);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c0 + j < cols) q[c0 + j] = static_cast<uint8_t>((j < 4 ? lo : hi) >> (8 * (j & 3)));
  }
}

// Sum of one value per lane, the same bits in every lane.
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum of h^2 and largest |u| of a row over its threads, the same bits in each.
// The order is fixed by the row's length (its number of threads), so a row's
// codes and scale do not depend on how many rows are with it, on strides or on
// alignment. `s_sum` and `s_max` alternate from call to call: one barrier each.
template <bool kNorm>
__device__ __forceinline__ void reduce_row(int lanes, float& sum, float big, uint32_t& most,
                                           float* s_sum, uint32_t* s_max) {
  most = __float_as_uint(big);
  if (lanes < 32) {  // several rows in a warp: each among its own lanes
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      if (o < lanes) {
        if constexpr (kNorm) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
      }
    }
    return;
  }
  if constexpr (kNorm) sum = warp_sum(sum);
  most = __reduce_max_sync(0xffffffffu, most);
  if (lanes == 32) return;
  const int lane = threadIdx.x & 31, warp = (threadIdx.x % lanes) >> 5, warps = lanes >> 5;
  if (lane == 0) {
    s_sum[warp] = sum;
    s_max[warp] = most;
  }
  __syncthreads();
  most = __reduce_max_sync(0xffffffffu, lane < warps ? s_max[lane] : 0u);
  if constexpr (kNorm) sum = warp_sum(lane < warps ? s_sum[lane] : 0.0f);
}

// A row from its reductions: its scale (stored by one thread) and its factor. In
// most / a the norm's r cancels, unless the row's maximum is the least there is.
template <bool kNorm, bool kE4M3>
__device__ __forceinline__ Factor finish_row(const RowsParams& p, int64_t row, float sum,
                                            uint32_t most, bool store) {
  constexpr float top = kE4M3 ? 448.0f : 127.0f;
  const float r = kNorm ? rsqrtf(fmaf(sum, p.inv_cols, p.eps)) : 1.0f;
  const float big = __uint_as_float(most) * r;
  const float a = fmaxf(big, kTiny);
  const bool bad = most >= kInfBits || !(a < __uint_as_float(kInfBits)) || (kNorm && !(r > 0.0f));
  if (store) p.scale[row] = bad ? __uint_as_float(0x7fc00000u) : a / top;
  const bool least = !(big > kTiny);
  const float by = least ? kTiny : __uint_as_float(most);
  Factor f;
  f.hi = top / by;
  f.lo = fmaf(-f.hi, by, top) * (f.hi * (1.0f / top));  // what is left of top, over by
  if (kNorm && least) {
    f.hi *= r;
    f.lo *= r;
  }
  if (bad) f = {0.0f, 0.0f};
  return f;
}

// Magnitudes above ~1e19 square past fp32's range, and h * weight may pass it where
// h * r * weight does not.
template <bool kNorm>
__device__ __forceinline__ bool past_range(float sum, uint32_t most) {
  return kNorm && (!(sum < __uint_as_float(kInfBits)) || most >= kInfBits);
}

// Such a row, from memory: its sum once more, of h * 2^-80 where the squares need it,
// then the maximum of y = h * r * weight itself, whose codes are made as the
// quantizer's. A true infinity or NaN stays one. The row's threads come here together
// (and with them the rows that share their warp, which are not `mine`); what was
// written of h is visible to them. An even number of reductions: the buffers'
// turn is the caller's again afterwards. (Compiled inline: as a called function it
// cost the rows that never come here a quarter of their time.)
template <typename T, bool kE4M3>
__device__ __forceinline__ void norm_past_range(const RowsParams& p, int64_t row, bool mine, float sum,
                                             float (*s_sum)[32], uint32_t (*s_max)[32],
                                             int parity) {
  const int lanes = p.lanes, t = threadIdx.x % lanes;
  const T* h = p.residual != nullptr ? static_cast<const T*>(p.h) + row * p.ldh
                                     : static_cast<const T*>(p.x) + row * p.ldx;
  auto values = [&](int c0, float factor, float (&u)[8], float& total) {
    load_row8<T>(h, c0, p.cols).values(u);
    float w[8];
    if (p.weight_f32)
      load_row8<float, true>(static_cast<const float*>(p.weight), c0, p.cols).values(w);
    else
      load_row8<T, true>(static_cast<const T*>(p.weight), c0, p.cols).values(w);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      u[j] *= factor;
      total = fmaf(u[j], u[j], total);
      u[j] *= w[j];
    }
  };
  float factor = sum < __uint_as_float(kInfBits) ? 1.0f : 8.271806125530277e-25f;  // 2^-80
  uint32_t most = 0;
#pragma unroll 1
  for (int turn = 0; turn < 2; ++turn) {
    float total = 0.0f, big = 0.0f;
#pragma unroll 1
    for (int c0 = t * 8; mine && c0 < p.cols; c0 += lanes * 8) {
      float u[8];
      values(c0, factor, u, total);
#pragma unroll
      for (int j = 0; j < 8; j += 2) big = max3_abs(big, u[j], u[j + 1]);
    }
    reduce_row<true>(lanes, total, big, most, s_sum[parity], s_max[parity]);
    parity ^= 1;
    if (turn == 0) factor *= rsqrtf(fmaf(total, p.inv_cols, p.eps * factor * factor));
  }
  if (!mine) return;
  const Factor f = finish_row<false, kE4M3>(p, row, 0.0f, most, t == 0);
#pragma unroll 1
  for (int c0 = t * 8; c0 < p.cols; c0 += lanes * 8) {
    float u[8] = {}, unused = 0.0f;
    if (f.hi != 0.0f) values(c0, factor, u, unused);
    store_codes<kE4M3, false>(p.q + row * p.ldq, c0, p.cols, p.codes_vec, u, f);
  }
}

__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void group_sync(int lanes) {
  if (lanes <= 32) __syncwarp();
  else __syncthreads();
}

// The eight values at byte `at` of a staged row.
template <typename T, bool kAligned>
__device__ __forceinline__ Eight<T> staged8(uint32_t at) {
  constexpr int kWords = Eight<T>::kWords;
  Eight<T> e;
  const int off = kAligned ? 0 : static_cast<int>(at & 15);
  uint32_t in[kWords + 4];
#pragma unroll
  for (int i = 0; i < kWords / 4 + (kAligned ? 0 : 1); ++i) {
    const uint4 v = lds_v4(at - off + 16 * i);
    in[4 * i] = v.x;
    in[4 * i + 1] = v.y;
    in[4 * i + 2] = v.z;
    in[4 * i + 3] = v.w;
  }
  if constexpr (kAligned) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) e.w[i] = in[i];
  } else {
    shift_any<kWords>(in, off, e.w);
  }
  return e;
}

// the quantizer; the norm without and with a residual
enum Mode : int { kCodes = 0, kNormed = 1, kSummed = 2 };

constexpr int kHold = 4;  // chunks of a row a thread holds as fp32

// Threads an SM holds of a kernel, hence the registers of one. The norm of whole
// rows spills at 64 registers and is faster with fewer threads of 80 (4096 x 8192
// 25.4 -> 22.5 us, 4096 x 5120 with a residual 28.3 -> 24.6; 16384 columns, one CTA
// an SM, 25.1 -> 26.0); the quantizer, whose long rows live from what is in flight,
// and the norm of other rows are not (codes 4096 x 28672 55 -> 62 us, norm 1000 x
// 5001 9.3 -> 9.9).
constexpr int sm_threads(Mode mode, bool whole, bool held) {
  return mode != kCodes && whole && held ? 768 : 1024;
}
constexpr int thread_regs(int threads) { return 65536 / threads / 8 * 8; }

// Rows staged in shared memory. A group of `lanes` threads walks its rows with
// `stages` of them in flight (cp.async): a thread copies the chunks it will
// read itself, so whole rows need no barrier but the reduction's; rows that
// start off a 16-byte boundary are copied as the aligned blocks that hold them
// (each holds at least one of their values) and shifted when they are read.
// Between the passes a thread holds u of its chunks (kHeld; rows of up to 16384
// columns) and its slot takes the next row at once (kEarly), or the first pass
// leaves h in the slot for the second.
//
// kWhole: every row of every operand is whole 16-byte chunks. It is a
// parameter of the kernel, not a test in it, because instructions set the
// pace: with the tests inside, and h and the weights read twice, a value cost
// 23 (codes) to 46 (norm with a residual) of them and the SMs issued at 70 % of
// their rate (4096 x 8192 with a residual 54.9 us).
template <typename T, Mode kMode, bool kE4M3, bool kWhole, bool kHeld>
__global__ void __maxnreg__(thread_regs(sm_threads(kMode, kWhole, kHeld)))
    rows8_staged_kernel(const __grid_constant__ RowsParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float s_sum[2][32];
  __shared__ uint32_t s_max[2][32];
  constexpr bool kNorm = kMode != kCodes;
  constexpr int kStreams = kMode == kSummed ? 2 : 1;
  constexpr int kSize = sizeof(T);
  constexpr bool kEarly = kWhole && kHeld;  // a slot is free once its row has been read
  // Chunks of a row that is not held whose loads go out together: the norm waits for
  // its weights' too (4096 x 20000 with a residual 134 us by twos, 129 by fours; int8
  // codes of 28672 columns 54.4 and 56.2).
  constexpr int kTurns = kNorm ? 4 : 2;
  const int lanes = p.lanes, groups = blockDim.x / lanes;
  const int group = threadIdx.x / lanes, t = threadIdx.x % lanes;
  // Rows and strides are 32 bits here (the launcher sees to it): an address is
  // one wide multiply-add where it is needed, not a register pair kept for it.
  const uint32_t step = gridDim.x * groups, first = blockIdx.x * groups + group;
  const uint32_t rows = static_cast<uint32_t>(p.rows);
  const uint32_t slots = smem_u32(smem) + group * p.stages * kStreams * p.slot;
  griddep_wait();
  griddep_launch_dependents();

  auto at = [](const void* base, uint32_t row, uint32_t stride) {
    return static_cast<const uint8_t*>(base) + static_cast<uint64_t>(row) * stride;
  };
  // distance of a stream's row from its 16-byte block
  auto offset = [&](const void* base, uint32_t row, uint32_t stride) {
    return kWhole ? 0 : static_cast<int>(reinterpret_cast<uintptr_t>(at(base, row, stride)) & 15);
  };
  auto copy_row = [&](const uint8_t* src, uint32_t slot) {
    const int bytes = p.cols * kSize;
    if constexpr (kEarly) {
      const uint8_t* s = src + t * 8 * kSize;
      uint32_t d = slot + t * 8 * kSize;
      const int stride = lanes * 8 * kSize;
#pragma unroll
      for (int c = 0; c < kHold; ++c, s += stride, d += stride)
        if ((c * lanes + t) * 8 < p.cols)
#pragma unroll
          for (int i = 0; i < kSize / 2; ++i) copy16_async(d + 16 * i, s + 16 * i);
    } else if constexpr (kWhole) {
      for (int b = t * 8 * kSize; b < bytes; b += lanes * 8 * kSize)
#pragma unroll
        for (int i = 0; i < kSize / 2; ++i) copy16_async(slot + b + 16 * i, src + b + 16 * i);
    } else {
      const int off = static_cast<int>(reinterpret_cast<uintptr_t>(src) & 15);
      for (int b = t * 16; b < off + bytes; b += lanes * 16) copy16_async(slot + b, src - off + b);
    }
  };
  auto fetch = [&](uint32_t row, int stage) {
    if (row < rows) {
      const uint32_t slot = slots + stage * kStreams * p.slot;
      copy_row(at(p.x, row, p.sx), slot);
      if constexpr (kMode == kSummed) copy_row(at(p.residual, row, p.sr), slot + p.slot);
    }
    copy_commit();
  };

  for (int s = 0; s + (kEarly ? 0 : 1) < p.stages; ++s) fetch(first + s * step, s);
  if constexpr (kNorm) {
    // the weights towards L1, where all rows of the SM read them: a thread a line
    // (one request a chunk and row group swamped the slices that hold them:
    // 16384 x 128 10.0 us)
    const int bytes = p.cols * (p.weight_f32 ? 4 : kSize);
    for (int b = threadIdx.x * 128; b < bytes; b += blockDim.x * 128)
      asm volatile("prefetch.global.L1 [%0];" ::"l"(static_cast<const uint8_t*>(p.weight) + b));
  }
  int stage = 0, parity = 0;
  // the same number of turns for every group of a CTA (a CTA has several only
  // when each is a warp or less, whose reduction needs no barrier)
  for (uint32_t base = blockIdx.x * groups; base < rows; base += step) {
    const uint32_t row = base + group;
    const bool live = row < rows;
    if constexpr (!kEarly)
      fetch(row + (p.stages - 1) * step, stage == 0 ? p.stages - 1 : stage - 1);
    if (p.stages == 1) copy_wait<0>();
    else if (p.stages == 2) copy_wait<1>();
    else copy_wait<3>();
    if constexpr (!kWhole) group_sync(lanes);
    const uint32_t slot = slots + stage * kStreams * p.slot;
    const int cols = live ? p.cols : 0;
    const int off = offset(p.x, row, p.sx);
    const int offr = kMode == kSummed ? offset(p.residual, row, p.sr) : 0;
    T* h = reinterpret_cast<T*>(const_cast<uint8_t*>(at(p.h, row, p.sh)));
    uint8_t* q = const_cast<uint8_t*>(at(p.q, row, p.sq));

    // h of the chunk at c0. First: the residual's addition, h stored (of a whole
    // row also left in its slot where it is read again; another adds again, and
    // in 16 bits is stored by store_shifted8).
    auto chunk = [&](int c0, auto start) {
      constexpr bool kStart = decltype(start)::value;
      Eight<T> e = staged8<T, kWhole>(slot + off + c0 * kSize);
      if constexpr (kMode == kSummed && (kStart || kHeld || !kWhole)) {
        add<T>(e, staged8<T, kWhole>(slot + p.slot + offr + c0 * kSize));
        if constexpr (kStart && kWhole) {
          store8<T>(h + c0, e);
          if constexpr (!kHeld) {
#pragma unroll
            for (int i = 0; i < Eight<T>::kWords / 4; ++i)
              sts_v4u(slot + c0 * kSize + 16 * i, e.w[4 * i], e.w[4 * i + 1], e.w[4 * i + 2],
                      e.w[4 * i + 3]);
          }
        } else if constexpr (kStart && kSize == 4) {
          store_row8<T>(h, c0, p.cols, e);
        }
      }
      return e;
    };
    // u = h * weight, the sum of h^2
    auto values = [&](const Eight<T>& e, int c0, float (&u)[8], float& sum) {
      e.values(u);
      if (!kWhole && c0 + 8 > p.cols) {  // the row's last chunk
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = c0 + j < p.cols ? u[j] : 0.0f;
      }
      if constexpr (kNorm) {
        float w[8];
        if (p.weight_f32)
          load_weights<float, kWhole>(static_cast<const float*>(p.weight), c0, p.cols).values(w);
        else
          load_weights<T, kWhole>(static_cast<const T*>(p.weight), c0, p.cols).values(w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          sum = fmaf(u[j], u[j], sum);
          u[j] *= w[j];
        }
      }
    };
    auto largest = [&](float big, const float (&u)[8]) {
#pragma unroll
      for (int j = 0; j < 8; j += 2) big = max3_abs(big, u[j], u[j + 1]);
      return big;
    };
    auto put = [&](int c0, const float (&u)[8], Factor f) {
      store_codes<kE4M3, kWhole>(q, c0, p.cols, p.codes_vec, u, f);
    };
    auto quantize = [&](Factor f) {  // from the staged row, or zeros
      if (kHeld || (kNorm && f.hi == 0.0f)) {
        const float zeros[8] = {};
#pragma unroll 1
        for (int c0 = t * 8; c0 < cols; c0 += lanes * 8) put(c0, zeros, f);
        return;
      }
#pragma unroll kTurns
      for (int c0 = t * 8; c0 < cols; c0 += lanes * 8) {
        float u[8] = {}, unused = 0.0f;
        if (kNorm || f.hi != 0.0f) values(chunk(c0, std::false_type{}), c0, u, unused);
        put(c0, u, f);
      }
    };

    float sum = 0.0f, big = 0.0f;
    uint32_t most;
    float held[kHeld ? kHold : 1][8];
    if constexpr (kHeld) {
#pragma unroll
      for (int c = 0; c < kHold; ++c) {
        const int c0 = (c * lanes + t) * 8;
        if constexpr (kMode == kSummed && !kWhole && kSize == 2) {
          if (c * lanes * 8 >= p.cols) break;  // (the same for the warp)
          Eight<T> e = {};
          if (c0 < cols) e = chunk(c0, std::true_type{});
          store_shifted8<T>(h, c0, cols, e, t == 0 || (t & 31) == 0,
                            t + 1 == lanes || (t & 31) == 31);
          if (c0 >= cols) continue;
          values(e, c0, held[c], sum);
          big = largest(big, held[c]);
        } else if (c0 < cols) {
          values(chunk(c0, std::true_type{}), c0, held[c], sum);
          big = largest(big, held[c]);
        }
      }
      if constexpr (kEarly) fetch(row + p.stages * step, stage);
    } else {
      // (whole chunks.) The quantizer takes the maximum of 16-bit values two at a time
      // as they lie: one instruction where unpacking them first took three (4096 x
      // 28672 57.1 -> 54.3 us; rows that are held have to be unpacked anyway).
      constexpr bool kPacked = !kNorm && kSize == 2;
      uint32_t big2 = 0;
#pragma unroll kTurns
      for (int c0 = t * 8; c0 < cols; c0 += lanes * 8) {
        const Eight<T> e = chunk(c0, std::true_type{});
        if constexpr (kPacked) {
#pragma unroll
          for (int i = 0; i < 4; ++i) big2 = max2_abs<T>(big2, e.w[i]);
        } else {
          values(e, c0, held[0], sum);
          big = largest(big, held[0]);
        }
      }
      if constexpr (kPacked) {
        float v[8];
        Eight<T>{big2, 0u, 0u, 0u}.values(v);
        big = max3_abs(0.0f, v[0], v[1]);
      }
    }
    reduce_row<kNorm>(lanes, sum, big, most, s_sum[parity], s_max[parity]);
    parity ^= 1;
    // a warp with several rows goes together
    const bool again = live && past_range<kNorm>(sum, most);
    if constexpr (kNorm) {
      if (lanes < 32 ? __any_sync(0xffffffffu, again) : again) {
        group_sync(lanes);  // threads may have stored values of h for one another
        norm_past_range<T, kE4M3>(p, row, again, sum, s_sum, s_max, parity);
      }
    }
    if (live && !again) {
      const Factor f = finish_row<kNorm, kE4M3>(p, row, sum, most, t == 0);
      if (!kHeld || f.hi == 0.0f) {
        quantize(f);
      } else {
#pragma unroll
        for (int c = 0; c < kHold; ++c) {
          const int c0 = (c * lanes + t) * 8;
          if (c0 < cols) put(c0, held[kHeld ? c : 0], f);
        }
      }
    }
    if constexpr (!kWhole) group_sync(lanes);  // the slot has been read by all
    stage = stage + 1 == p.stages ? 0 : stage + 1;
  }
  copy_wait<0>();
}

// Rows of which the stages do not fit shared memory, rows of more than 16384
// columns that are not whole 16-byte chunks, and rows 4 GB or more apart: one CTA
// a row, read again, from L2, for the codes. The row's threads and the order of its
// sum are those of the staged kernel, whatever its width: a CTA of `lanes` threads,
// or one warp of which `lanes` hold the row and the rest hold nothing.
template <typename T, bool kNorm, bool kE4M3>
__global__ void __launch_bounds__(kMaxLanes) rows8_long_kernel(const __grid_constant__ RowsParams p) {
  __shared__ float s_sum[2][32];
  __shared__ uint32_t s_max[2][32];
  const int64_t row = blockIdx.x;
  const int t = threadIdx.x, lanes = p.lanes;
  const int begin = t < lanes ? t * 8 : p.cols;
  griddep_wait();
  griddep_launch_dependents();
  const T* x = static_cast<const T*>(p.x) + row * p.ldx;
  const T* r = static_cast<const T*>(p.residual) + row * p.ldr;
  T* h = static_cast<T*>(p.h) + row * p.ldh;
  const bool residual = kNorm && p.residual != nullptr;
  auto values = [&](bool start, int c0, float (&u)[8], float& sum) {
    Eight<T> e = load_row8<T>(residual && !start ? h : x, c0, p.cols);
    if (residual && start) {
      add<T>(e, load_row8<T>(r, c0, p.cols));
      store_row8<T>(h, c0, p.cols, e);
    }
    e.values(u);
    if constexpr (kNorm) {
      float w[8];
      if (p.weight_f32)
        load_row8<float, true>(static_cast<const float*>(p.weight), c0, p.cols).values(w);
      else
        load_row8<T, true>(static_cast<const T*>(p.weight), c0, p.cols).values(w);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sum = fmaf(u[j], u[j], sum);
        u[j] *= w[j];
      }
    }
  };
  float sum = 0.0f, big = 0.0f;
  uint32_t most;
  for (int c0 = begin; c0 < p.cols; c0 += lanes * 8) {
    float u[8];
    values(true, c0, u, sum);
#pragma unroll
    for (int j = 0; j < 8; j += 2) big = max3_abs(big, u[j], u[j + 1]);
  }
  reduce_row<kNorm>(lanes, sum, big, most, s_sum[0], s_max[0]);
  if constexpr (kNorm) {
    bool again = past_range<kNorm>(sum, most);
    if (lanes < 32) again = __any_sync(0xffffffffu, again);  // the whole warp as the row
    if (again) {
      norm_past_range<T, kE4M3>(p, row, t < lanes, sum, s_sum, s_max, 1);
      return;
    }
  }
  const Factor f = finish_row<kNorm, kE4M3>(p, row, sum, most, t == 0);
  for (int c0 = begin; c0 < p.cols; c0 += lanes * 8) {
    float u[8], unused = 0.0f;
    values(false, c0, u, unused);
    if (f.hi == 0.0f) {
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = 0.0f;
    }
    store_codes<kE4M3, false>(p.q + row * p.ldq, c0, p.cols, p.codes_vec, u, f);
  }
}

// Eight codes (two words) times the row's scale. An int8 code becomes a float by
// byte selection: with its sign bit flipped it is the low byte of 2^23 + 128 +
// code, whose excess one exact subtraction takes off (the conversion
// instruction runs at a quarter of their rate).
template <typename T, bool kE4M3>
__device__ __forceinline__ Eight<T> code_values(uint32_t w0, uint32_t w1, float s) {
  float v[8];
  if constexpr (kE4M3) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const uint32_t pair = (j < 4 ? w0 : w1) >> (8 * (j & 2));
      const __half2 h(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(pair & 0xffffu),
                                                 __NV_E4M3));
      const float2 f = __half22float2(h);
      v[j] = f.x * s;
      v[j + 1] = f.y * s;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t flipped = (j < 4 ? w0 : w1) ^ 0x80808080u;
      v[j] = (__uint_as_float(prmt(flipped, 0x4b000000u, 0x7540 | (j & 3))) - 8388736.0f) * s;
    }
  }
  Eight<T> e;
  e.round(v);
  return e;
}

// kWhole: 32 bytes of values a thread (eight codes to fp32, sixteen to 16 bits).
// Else eight: rows of values that start off a 16-byte boundary (odd widths)
// begin with up to seven single values (item 0), so that the chunks after them
// store whole; their codes then start at any byte, and come from the words that
// hold them (1000 x 5001: 5.7 us, by bytes 21.5).
template <typename T, bool kE4M3, bool kWhole>
__global__ void __launch_bounds__(256)
    dequantize_rows_kernel(const uint8_t* q, int64_t ldq, const float* scale, T* out, int64_t ldo,
                           int64_t rows, int cols) {
  constexpr int kPer = sizeof(T) == 4 ? 8 : 16;
  griddep_wait();
  griddep_launch_dependents();
  const int item = blockIdx.x * blockDim.x + threadIdx.x;
  for (int64_t row = static_cast<int64_t>(blockIdx.y) * blockDim.y + threadIdx.y; row < rows;
       row += static_cast<int64_t>(gridDim.y) * blockDim.y) {
    const uint8_t* src = q + row * ldq;
    T* dst = out + row * ldo;
    if constexpr (kWhole) {
      const int c0 = item * kPer;
      if (c0 >= cols) continue;
      const float s = scale[row];
      if constexpr (kPer == 8) {
        const uint2 w = __ldcg(reinterpret_cast<const uint2*>(src + c0));
        store8<T>(dst + c0, code_values<T, kE4M3>(w.x, w.y, s));
      } else {
        const uint4 w = __ldcg(reinterpret_cast<const uint4*>(src + c0));
        store8<T>(dst + c0, code_values<T, kE4M3>(w.x, w.y, s));
        store8<T>(dst + c0 + 8, code_values<T, kE4M3>(w.z, w.w, s));
      }
      continue;
    }
    const int head =
        static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(dst) & 15)) & 15) / sizeof(T));
    const int c0 = head == 0 ? item * 8 : item == 0 ? 0 : head + (item - 1) * 8;
    const int c1 = min(cols, head != 0 && item == 0 ? head : c0 + 8);
    if (c0 >= c1) continue;
    const float s = scale[row];
    uint32_t w[2] = {0u, 0u};
    if (c1 - c0 == 8) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(src + c0);
      const uint32_t* base = reinterpret_cast<const uint32_t*>(at & ~static_cast<uintptr_t>(3));
      const int bits = static_cast<int>(at & 3) * 8;
      const uint32_t a = __ldcg(base), b = __ldcg(base + 1);
      const uint32_t c = bits != 0 ? __ldcg(base + 2) : 0u;
      w[0] = __funnelshift_r(a, b, bits);
      w[1] = __funnelshift_r(b, c, bits);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c0 + j < c1) w[j >> 2] |= static_cast<uint32_t>(src[c0 + j]) << (8 * (j & 3));
    }
    const Eight<T> e = code_values<T, kE4M3>(w[0], w[1], s);
    if (c1 - c0 == 8) {
      store8<T>(dst + c0, e);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c0 + j < c1) dst[c0 + j] = e.element(j);
    }
  }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <typename... P, typename... A>
cudaError_t launch_chained(void (*kernel)(P...), dim3 grid, dim3 block, int smem, cudaStream_t s,
                           A... args) {
  if (smem > 40 * 1024) {  // 48 KB less the static arrays need no attribute
    const cudaError_t e = set_max_smem(reinterpret_cast<const void*>(kernel), kMostStaged);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

template <typename T, Mode kMode, bool kE4M3>
cudaError_t launch_staged(const RowsParams& p, bool whole, dim3 grid, int threads, int smem,
                          cudaStream_t s) {
  if (!whole)
    return launch_chained(rows8_staged_kernel<T, kMode, kE4M3, false, true>, grid, threads, smem, s, p);
  if (p.cols <= kHold * 8 * kMaxLanes)
    return launch_chained(rows8_staged_kernel<T, kMode, kE4M3, true, true>, grid, threads, smem, s, p);
  return launch_chained(rows8_staged_kernel<T, kMode, kE4M3, true, false>, grid, threads, smem, s, p);
}

template <typename T, bool kE4M3>
cudaError_t launch_mode(const RowsParams& p, bool norm, bool whole, bool staged, int threads,
                        int grid, int smem, cudaStream_t s) {
  if (!staged) {
    const int block = std::max(p.lanes, 32);
    return norm ? launch_chained(rows8_long_kernel<T, true, kE4M3>, grid, block, 0, s, p)
                : launch_chained(rows8_long_kernel<T, false, kE4M3>, grid, block, 0, s, p);
  }
  if (!norm) return launch_staged<T, kCodes, kE4M3>(p, whole, grid, threads, smem, s);
  return p.residual != nullptr ? launch_staged<T, kSummed, kE4M3>(p, whole, grid, threads, smem, s)
                               : launch_staged<T, kNormed, kE4M3>(p, whole, grid, threads, smem, s);
}

// Threads per row: four chunks of eight columns each, from 4 up to kMaxLanes; a
// function of the row's length alone (it fixes the order of the sum). With two
// chunks the per-row work of twice as many warps costs more than it hides (8192
// x 4096 codes 28.8 us, with four 15.7). Rows of up to 1024 columns are a
// warp's or a part of it, several to a CTA (a warp each: 100000 x 128 22.4 us).
// Rows in flight: two, four of such short ones; the grid is what fits the SMs at
// once.
template <typename T>
cudaError_t launch_rows(RowsParams p, bool norm, cudaStream_t s) {
  constexpr int kSize = sizeof(T);
  p.lanes = 4;
  while (p.lanes < kMaxLanes && p.lanes * 32 < p.cols) p.lanes *= 2;
  p.inv_cols = 1.0f / static_cast<float>(p.cols);
  const bool residual = norm && p.residual != nullptr;
  const auto whole = [](const void* b, int64_t ld) {
    return aligned16(b) && (ld * kSize) % 16 == 0;
  };
  p.codes_vec = (reinterpret_cast<uintptr_t>(p.q) & 7) == 0 && p.ldq % 8 == 0;
  const bool chunks = p.cols % 8 == 0 && p.codes_vec && whole(p.x, p.ldx) &&
                      (!residual || (whole(p.residual, p.ldr) && whole(p.h, p.ldh))) &&
                      (!norm || aligned16(p.weight));

  const int threads = p.lanes <= 32 ? 128 : p.lanes;
  const int groups = threads / p.lanes;
  // a chunk past an unaligned row's last block is read (and discarded)
  const int64_t cols8 = static_cast<int64_t>(p.cols + 7) / 8 * 8;
  const int64_t slot = cols8 * kSize + (chunks ? 0 : 32);
  const int64_t streams = residual ? 2 : 1;
  p.stages = p.lanes <= 32 ? 4 : 2;
  const bool held = !chunks || p.cols <= kHold * 8 * kMaxLanes;
  const int resident =
      sm_threads(!norm ? kCodes : residual ? kSummed : kNormed, chunks, held) / threads;
  if (chunks && held && p.lanes > 32 && (slot * streams * 2 + 1536) * resident > 228 * 1024)
    p.stages = 1;  // as many CTAs as the registers allow before a second row in flight
  const int64_t bytes = slot * streams * groups * p.stages;
  const int64_t widest = std::max({p.ldx, p.ldr, p.ldh, p.ldq}) * kSize;
  p.sx = static_cast<uint32_t>(p.ldx * kSize);
  p.sr = static_cast<uint32_t>(p.ldr * kSize);
  p.sh = static_cast<uint32_t>(p.ldh * kSize);
  p.sq = static_cast<uint32_t>(p.ldq);
  const bool staged = bytes <= kMostStaged && widest < (1ll << 32) &&
                      (chunks || p.cols <= kHold * 8 * kMaxLanes);
  p.slot = static_cast<int>(staged ? slot : 0);
  const int64_t per_sm =
      std::max<int64_t>(1, std::min<int64_t>(resident, 228 * 1024 / (bytes + 1536)));
  const int64_t ctas = (p.rows + groups - 1) / groups;
  const int grid =
      static_cast<int>(staged ? std::min<int64_t>(ctas, per_sm * num_sms()) : p.rows);
  const int smem = static_cast<int>(staged ? bytes : 0);
  return p.e4m3 ? launch_mode<T, true>(p, norm, chunks, staged, threads, grid, smem, s)
                : launch_mode<T, false>(p, norm, chunks, staged, threads, grid, smem, s);
}

cudaError_t launch_rows_any(const RowsParams& p, int dtype, bool norm, cudaStream_t s) {
  switch (dtype) {
    case PK_F16: return launch_rows<__half>(p, norm, s);
    case PK_BF16: return launch_rows<__nv_bfloat16>(p, norm, s);
    case PK_F32: return launch_rows<float>(p, norm, s);
    default: return cudaErrorInvalidValue;
  }
}

template <typename T>
cudaError_t launch_dequantize_typed(const uint8_t* q, int64_t ldq, const float* scale, T* out,
                                    int64_t ldo, int64_t rows, int cols, int e4m3,
                                    cudaStream_t s) {
  const bool whole = cols % 16 == 0 && aligned16(q) && ldq % 16 == 0 && aligned16(out) &&
                     (ldo * sizeof(T)) % 16 == 0;
  // one item more for the start of an unaligned row
  const int items = whole ? cols / (sizeof(T) == 4 ? 8 : 16) : (cols + 7) / 8 + 1;
  int tx = 32;
  while (tx < 256 && tx < items) tx *= 2;
  const int ty = 256 / tx;
  const int64_t gy = (rows + ty - 1) / ty;
  const dim3 grid(static_cast<unsigned>((items + tx - 1) / tx),
                  static_cast<unsigned>(gy < 65535 ? gy : 65535));
  const dim3 block(tx, ty);
  auto go = [&](auto kernel) {
    return launch_chained(kernel, grid, block, 0, s, q, ldq, scale, out, ldo, rows, cols);
  };
  if (e4m3)
    return whole ? go(dequantize_rows_kernel<T, true, true>) : go(dequantize_rows_kernel<T, true, false>);
  return whole ? go(dequantize_rows_kernel<T, false, true>) : go(dequantize_rows_kernel<T, false, false>);
}

}  // namespace

cudaError_t launch_quantize_rows(const void* x, int dtype, int64_t rows, int64_t cols, int64_t ldx,
                                 void* q, bool e4m3, int64_t ldq, float* scale, cudaStream_t s) {
  RowsParams p{};
  p.x = x;
  p.ldx = ldx;
  p.q = static_cast<uint8_t*>(q);
  p.ldq = ldq;
  p.scale = scale;
  p.rows = rows;
  p.cols = static_cast<int>(cols);
  p.e4m3 = e4m3;
  return launch_rows_any(p, dtype, false, s);
}

cudaError_t launch_rms_norm_quant(const void* x, int dtype, int64_t rows, int64_t cols,
                                  int64_t ldx, const void* residual, int64_t ldr,
                                  const void* weight, bool weight_f32, float eps, void* h,
                                  int64_t ldh, void* q, bool e4m3, int64_t ldq, float* scale,
                                  cudaStream_t s) {
  RowsParams p{};
  p.x = x;
  p.ldx = ldx;
  p.residual = residual;
  p.ldr = ldr;
  p.weight = weight;
  p.weight_f32 = weight_f32;
  p.eps = eps;
  p.h = h;
  p.ldh = ldh;
  p.q = static_cast<uint8_t*>(q);
  p.ldq = ldq;
  p.scale = scale;
  p.rows = rows;
  p.cols = static_cast<int>(cols);
  p.e4m3 = e4m3;
  return launch_rows_any(p, dtype, true, s);
}

cudaError_t launch_dequantize_rows(const void* q, bool e4m3, int64_t rows, int64_t cols,
                                   int64_t ldq, const float* scale, void* out, int out_dtype,
                                   int64_t ldo, cudaStream_t s) {
  const uint8_t* b = static_cast<const uint8_t*>(q);
  const int n = static_cast<int>(cols);
  switch (out_dtype) {
    case PK_F16:
      return launch_dequantize_typed(b, ldq, scale, static_cast<__half*>(out), ldo, rows, n, e4m3, s);
    case PK_BF16:
      return launch_dequantize_typed(b, ldq, scale, static_cast<__nv_bfloat16*>(out), ldo, rows, n,
                                     e4m3, s);
    case PK_F32:
      return launch_dequantize_typed(b, ldq, scale, static_cast<float*>(out), ldo, rows, n, e4m3, s);
    default: return cudaErrorInvalidValue;
  }
}

}  // namespace pk
