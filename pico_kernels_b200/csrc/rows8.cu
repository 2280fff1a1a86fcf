// Rows in 8 bits: the quantizer of activations and weights with one scale per
// row, its inverse, and the RMS norm that writes its output already quantized.
//
//   quantize      a = max(max_k |x_k|, 1e-12),  scale = a / most,
//                 q_k = round(x_k * (most / a)),  most = 127 (int8) or 448 (e4m3)
//   rms norm      h = T(x + residual),  r = 1 / sqrt(mean(h^2) + eps),
//                 y_k = h_k * r * w_k, quantized as above
//   dequantize    x_k = q_k * scale
//
// All three are bound by HBM: a row is read once, kept in registers while its
// sum and its largest magnitude are reduced, and written once. The norm needs
// one reduction, not two (the sum for r, then the maximum of y): r multiplies
// the whole row, so the codes of y are those of u_k = h_k * w_k, and the sum of
// h^2 and the maximum of |u| are reduced together; r enters the scale alone.
// The maximum propagates NaN (across threads on the bit patterns of |u|, ordered
// like the values with infinities and NaN on top), so none can be lost in it.
//
// A row that holds a NaN or an infinity has no 8-bit form: it gets scale NaN
// and codes 0, so that every product with it is NaN and no other row is
// touched. Sums, maxima and scales are fp32; the only roundings to fewer bits
// are the stored h (the residual stream's own type, which is what the next
// layer adds to, so the norm is that of the stored value) and the codes.
#include <cuda_fp8.h>

#include <type_traits>

#include "pk_common.cuh"

namespace pk {
namespace {

constexpr float kTiny = 1e-12f;     // smallest row maximum, as in the int4 group scales
constexpr uint32_t kInfBits = 0x7f800000u;
// Threads of a CTA by chunks held, and the CTAs of an SM the registers are
// kept to.
constexpr int max_threads(int chunks) { return chunks >= 4 ? 512 : 1024; }
#ifndef MINB4
#define MINB4 2
#endif
#ifndef MINB8
#define MINB8 2
#endif
constexpr int min_ctas(int chunks) { return chunks == 4 ? MINB4 : chunks == 8 ? MINB8 : 1; }
constexpr int kRowWarps = 8;        // rows per CTA when a warp holds a row

struct RowsParams {
  const void* x;
  const void* residual;  // norm: added to x (nullptr: none)
  const void* weight;    // norm: fp32, or x's type
  void* h;               // norm with a residual: the sum, in x's type
  uint8_t* q;
  float* scale;
  int64_t ldx, ldr, ldh, ldq;
  int64_t rows;
  int cols;
  int lanes;             // threads of a row
  int weight_f32;
  int codes_vec;         // rows of codes 8-byte aligned
  int e4m3;
  float eps;
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
// norm's weights (kept in L1: every row of the SM reads them).
template <bool kWeights>
__device__ __forceinline__ uint4 load16(const uint4* p) {
  return kWeights ? __ldg(p) : __ldcg(p);
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
  const int bits = (off & 3) * 8;
  Eight<T> e;
  switch (off >> 2) {
    case 0: shift_words<kWords, 0>(in, bits, e.w); break;
    case 1: shift_words<kWords, 1>(in, bits, e.w); break;
    case 2: shift_words<kWords, 2>(in, bits, e.w); break;
    default: shift_words<kWords, 3>(in, bits, e.w); break;
  }
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
template <typename T, bool kVec, bool kWeights = false>
__device__ __forceinline__ Eight<T> load_row8(const T* row, int c0, int cols) {
  if (c0 + 8 <= cols)
    return kVec ? load8<T, kWeights>(row + c0) : load8_shifted<T, kWeights>(row + c0);
  Eight<T> e;
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = c0 + j < cols ? as_f32<T>(row[c0 + j]) : 0.0f;
  e.round(v);  // the values themselves
  return e;
}

// The row's h at column c0 in its own type: x, or in a later pass over a row
// with a residual the sum the thread itself has stored.
template <typename T, bool kNorm, bool kVec>
__device__ __forceinline__ Eight<T> load_h(const RowsParams& p, int64_t row, int c0, bool first) {
  if (kNorm && p.residual != nullptr && !first)
    return load_row8<T, kVec>(static_cast<const T*>(p.h) + row * p.ldh, c0, p.cols);
  return load_row8<T, kVec>(static_cast<const T*>(p.x) + row * p.ldx, c0, p.cols);
}

// h = x + residual, stored.
template <typename T, bool kVec>
__device__ __forceinline__ void add_residual(const RowsParams& p, int64_t row, int c0,
                                             const Eight<T>& r, Eight<T>& e) {
  T* h = static_cast<T*>(p.h) + row * p.ldh + c0;
  float a[8], b[8];
  e.values(a);
  r.values(b);
#pragma unroll
  for (int j = 0; j < 8; ++j) a[j] += b[j];
  e.round(a);
  if (kVec && c0 + 8 <= p.cols) {
    store8<T>(h, e);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c0 + j < p.cols) h[j] = e.element(j);
  }
}

// u = h * factor * weight of a chunk, the sum of (h * factor)^2 in `sum`. The
// weights are read again for the codes (from L1 or L2) rather than u kept: a
// held chunk is then 16 bytes a thread of a 16-bit type, not 32.
template <typename T, bool kNorm, bool kVec>
__device__ __forceinline__ void values(const RowsParams& p, const Eight<T>& e, int c0,
                                       float factor, float (&u)[8], float& sum) {
  e.values(u);
  if constexpr (kNorm) {
    sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      u[j] *= factor;
      sum = fmaf(u[j], u[j], sum);
    }
    float w[8];
    if (p.weight_f32)
      load_row8<float, kVec, true>(static_cast<const float*>(p.weight), c0, p.cols).values(w);
    else
      load_row8<T, kVec, true>(static_cast<const T*>(p.weight), c0, p.cols).values(w);
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] *= w[j];
  }
}

// Four int8 codes of u * f: adding 1.5 * 2^23 leaves the product, rounded half
// to even by the addition (fused: one rounding), as an integer in the low bits.
// |u * f| is at most 127 and a few last places, so no code passes 127. One
// multiply-add a value and three byte selections, where conversions, clamps and
// shifts took eight instructions.
__device__ __forceinline__ uint32_t int8_codes4(const float* u, float f) {
  constexpr float kMagic = 12582912.0f;
  uint32_t b[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) b[j] = __float_as_uint(fmaf(u[j], f, kMagic));
  return prmt(prmt(b[0], b[1], 0x0040), prmt(b[2], b[3], 0x0040), 0x5410);
}

// Largest of |a|, |b|, |c|; NaN if one is NaN.
__device__ __forceinline__ float max3_abs(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(fabsf(b)), "f"(fabsf(c)));
  return r;
}

// Codes of the chunk at column c0. Rows of codes are 8-byte aligned on every
// path the launcher calls vector; elsewhere (a caller's own pitch) by bytes.
__device__ __forceinline__ void store_codes(const RowsParams& p, int64_t row, int c0,
                                            const float (&u)[8], float f) {
  uint8_t* q = p.q + row * p.ldq + c0;
  const bool e4m3 = p.e4m3 != 0;
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (e4m3) {
      const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(u[4 * i] * f, u[4 * i + 1] * f),
                                                   __NV_SATFINITE, __NV_E4M3);
      const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(u[4 * i + 2] * f, u[4 * i + 3] * f),
                                                   __NV_SATFINITE, __NV_E4M3);
      w[i] = lo | (hi << 16);
    } else {
      w[i] = int8_codes4(u + 4 * i, f);
    }
  }
  if (p.codes_vec && c0 + 8 <= p.cols) {
    *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (c0 + j < p.cols) q[j] = static_cast<uint8_t>(w[j >> 2] >> (8 * (j & 3)));
  }
}

// Sum of one value per lane, the same bits in every lane.
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

constexpr int kBlocks = 128;  // sums of 256 columns in a held row (32768 columns)

// kChunks chunks of eight values per thread stay in registers; kChunks = 0
// (rows of more than 32768 columns) reads the row again, from L2, instead.
//
// The sum is the same tree whatever the number of threads: eight columns in
// order, 32 such chunks (a block of 256 columns) by a warp's shuffles, blocks
// 32 apart in order, those 32 sums by shuffles. So a row's codes and scale do
// not depend on how many rows are with it, on strides or on alignment.
template <typename T, bool kNorm, int kChunks, bool kVec>
__global__ void __launch_bounds__(max_threads(kChunks), min_ctas(kChunks)) rows8_kernel(const RowsParams p) {
  __shared__ float s_sum[kBlocks];
  __shared__ uint32_t s_max[32];
  const int lanes = p.lanes;
  const int t = threadIdx.x % lanes;
  const int lane = threadIdx.x & 31, warps = lanes >> 5, warp = t >> 5;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (blockDim.x / lanes) + threadIdx.x / lanes;
  griddep_wait();
  griddep_launch_dependents();
  if (row >= p.rows) return;  // whole warps: a CTA with several rows has one per warp

  constexpr int kHeld = kChunks > 0 ? kChunks : 1;
  const int chunks = kChunks > 0 ? kChunks : (p.cols + lanes * 8 - 1) / (lanes * 8);
  Eight<T> held[kHeld];
  if constexpr (kChunks > 0) {
    // every load of the row before its first store: h may be x or residual, so
    // a store between them would hold the later loads back
#pragma unroll
    for (int c = 0; c < kChunks; ++c)
      held[c] = load_h<T, kNorm, kVec>(p, row, (c * lanes + t) * 8, true);
    if (kNorm && p.residual != nullptr) {
      Eight<T> r[kHeld];
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
        r[c] = load_row8<T, kVec>(static_cast<const T*>(p.residual) + row * p.ldr,
                                  (c * lanes + t) * 8, p.cols);
#pragma unroll
      for (int c = 0; c < kChunks; ++c)
        add_residual<T, kVec>(p, row, (c * lanes + t) * 8, r[c], held[c]);
    }
  }
  float sum = 0.0f;
  uint32_t most = 0u;
  auto pass = [&](bool first, float factor) {
    float mine = 0.0f;  // one-warp rows: lane c holds block c; long rows: this warp's blocks
    float big = 0.0f;
    if (warps > 1) __syncthreads();  // an earlier pass has read s_sum
#pragma unroll(kHeld)
    for (int c = 0; c < (kChunks > 0 ? kChunks : chunks); ++c) {
      const int c0 = (c * lanes + t) * 8;
      if constexpr (kChunks == 0) {
        held[0] = load_h<T, kNorm, kVec>(p, row, c0, first);
        if (kNorm && p.residual != nullptr && first)
          add_residual<T, kVec>(
              p, row, c0,
              load_row8<T, kVec>(static_cast<const T*>(p.residual) + row * p.ldr, c0, p.cols),
              held[0]);
      }
      float u[8], s8 = 0.0f;
      values<T, kNorm, kVec>(p, held[kChunks > 0 ? c : 0], c0, factor, u, s8);
#pragma unroll
      for (int j = 0; j < 8; j += 2) big = max3_abs(big, u[j], u[j + 1]);
      if constexpr (kNorm) {
        s8 = warp_sum(s8);
        if constexpr (kChunks == 0) {
          mine += s8;
        } else if (warps == 1) {
          if (lane == c) mine = s8;
        } else if (lane == 0) {
          s_sum[c * warps + warp] = s8;
        }
      }
    }
    most = __reduce_max_sync(0xffffffffu, __float_as_uint(big));
    if (warps > 1) {
      if (lane == 0) {
        s_max[warp] = most;
        if (kNorm && kChunks == 0) s_sum[warp] = mine;
      }
      __syncthreads();
      most = __reduce_max_sync(0xffffffffu, lane < warps ? s_max[lane] : 0u);
      if constexpr (kNorm) {
        const int blocks = kHeld * warps;
        mine = 0.0f;
        for (int b = lane; b < blocks; b += 32) mine += s_sum[b];
      }
    }
    if constexpr (kNorm) sum = warp_sum(mine);
  };
  pass(true, 1.0f);
  float factor = 1.0f;
  if (kNorm && (!(sum < __uint_as_float(kInfBits)) || most >= kInfBits)) {
    // Magnitudes above ~1e19 square past fp32's range: once more on h * 2^-80,
    // which cancels in the norm (eps does not reach such sums). A true
    // infinity or NaN stays one.
    factor = 8.271806125530277e-25f;  // 2^-80
    pass(false, factor);
  }

  const float top = p.e4m3 ? 448.0f : 127.0f;
  const float eps = factor == 1.0f ? p.eps : 0.0f;
  const float r = kNorm ? 1.0f / sqrtf(sum / static_cast<float>(p.cols) + eps) : 1.0f;
  const float a = fmaxf(__uint_as_float(most) * r, kTiny);
  const bool bad = most >= kInfBits || !(a < __uint_as_float(kInfBits)) || (kNorm && !(r > 0.0f));
  const float f = kNorm ? r * (top / a) : top / a;
  if (t == 0) p.scale[row] = bad ? __uint_as_float(0x7fc00000u) : a / top;
#pragma unroll(kHeld)
  for (int c = 0; c < (kChunks > 0 ? kChunks : chunks); ++c) {
    const int c0 = (c * lanes + t) * 8;
    if constexpr (kChunks == 0) held[0] = load_h<T, kNorm, kVec>(p, row, c0, false);
    float u[8], unused;
    values<T, kNorm, kVec>(p, held[kChunks > 0 ? c : 0], c0, factor, u, unused);
    if (bad) {
#pragma unroll
      for (int j = 0; j < 8; ++j) u[j] = 0.0f;
    }
    store_codes(p, row, c0, u, bad ? 0.0f : f);
  }
}

// Eight codes a thread: one 8-byte load, 16 or 32 bytes of values. Rows of
// values that start off a 16-byte boundary (odd widths) begin with up to seven
// single values (item 0), so that the chunks after them store whole; their
// codes then start at any byte, and come from the two words that hold them.
template <typename T>
__global__ void __launch_bounds__(256)
    dequantize_rows_kernel(const uint8_t* __restrict__ q, int64_t ldq,
                           const float* __restrict__ scale, T* __restrict__ out, int64_t ldo,
                           int64_t rows, int cols, int e4m3) {
  griddep_wait();
  griddep_launch_dependents();
  const int item = blockIdx.x * blockDim.x + threadIdx.x;
  for (int64_t row = static_cast<int64_t>(blockIdx.y) * blockDim.y + threadIdx.y; row < rows;
       row += static_cast<int64_t>(gridDim.y) * blockDim.y) {
    const uint8_t* src = q + row * ldq;
    T* dst = out + row * ldo;
    const float s = scale[row];
    const int head = static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(dst) & 15)) & 15) / sizeof(T));
    const int c0 = head == 0 ? item * 8 : item == 0 ? 0 : head + (item - 1) * 8;
    const int c1 = min(cols, head != 0 && item == 0 ? head : c0 + 8);
    if (c0 >= c1) continue;
    uint32_t w[2] = {0u, 0u};
    if (c1 - c0 == 8) {
      const uintptr_t at = reinterpret_cast<uintptr_t>(src + c0);
      const uint32_t* base = reinterpret_cast<const uint32_t*>(at & ~static_cast<uintptr_t>(3));
      const int bits = static_cast<int>(at & 3) * 8;
      if ((at & 7) == 0) {
        const uint2 v = __ldcg(reinterpret_cast<const uint2*>(at));
        w[0] = v.x;
        w[1] = v.y;
      } else {
        const uint32_t a = __ldcg(base), b = __ldcg(base + 1);
        const uint32_t c = bits != 0 ? __ldcg(base + 2) : 0u;
        w[0] = __funnelshift_r(a, b, bits);
        w[1] = __funnelshift_r(b, c, bits);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (c0 + j < c1) w[j >> 2] |= static_cast<uint32_t>(src[c0 + j]) << (8 * (j & 3));
    }
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      const uint32_t pair = w[j >> 2] >> (8 * (j & 2));
      if (e4m3) {
        const __half2 h(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(pair & 0xffffu),
                                                   __NV_E4M3));
        const float2 f = __half22float2(h);
        v[j] = f.x * s;
        v[j + 1] = f.y * s;
      } else {
        v[j] = static_cast<float>(static_cast<int8_t>(pair)) * s;
        v[j + 1] = static_cast<float>(static_cast<int8_t>(pair >> 8)) * s;
      }
    }
    Eight<T> e;
    e.round(v);
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
cudaError_t launch_chained(void (*kernel)(P...), dim3 grid, dim3 block, cudaStream_t s, A... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

// Threads per row and chunks per thread. A row of up to 1024 columns is one
// warp's, eight rows to a CTA (no shared memory, no barrier); a longer row is a
// CTA's. Few rows (decode) spread each row over as many threads as it has
// chunks, for the shortest chain of loads.
template <typename T, bool kNorm, bool kVec>
cudaError_t launch_rows(RowsParams p, cudaStream_t s) {
  const int items = (p.cols + 7) / 8;
  const int per_lane = p.rows <= num_sms() ? 1 : 4;
  int lanes = 32;
  while (lanes < 1024 && lanes * per_lane < items) lanes *= 2;
  if (items > 2 * 1024 && items <= 8 * 512) lanes = 512;
  p.lanes = lanes;
  const int chunks = (items + lanes - 1) / lanes;
  const int threads = lanes == 32 ? 32 * kRowWarps : lanes;
  const int64_t per_cta = threads / lanes;
  const dim3 grid(static_cast<unsigned>((p.rows + per_cta - 1) / per_cta));
  if (items > 8 * 512) return launch_chained(rows8_kernel<T, kNorm, 0, kVec>, grid, threads, s, p);
  if (chunks <= 1) return launch_chained(rows8_kernel<T, kNorm, 1, kVec>, grid, threads, s, p);
  if (chunks <= 2) return launch_chained(rows8_kernel<T, kNorm, 2, kVec>, grid, threads, s, p);
  if (chunks <= 4) return launch_chained(rows8_kernel<T, kNorm, 4, kVec>, grid, threads, s, p);
  return launch_chained(rows8_kernel<T, kNorm, 8, kVec>, grid, threads, s, p);
}

template <typename T>
cudaError_t launch_rows_typed(RowsParams p, bool norm, cudaStream_t s) {
  const auto whole = [](const void* b, int64_t ld, int64_t size) {
    return aligned16(b) && (ld * size) % 16 == 0;
  };
  const bool vec = whole(p.x, p.ldx, sizeof(T)) &&
                   (p.residual == nullptr ||
                    (whole(p.residual, p.ldr, sizeof(T)) && whole(p.h, p.ldh, sizeof(T)))) &&
                   (!norm || aligned16(p.weight));
  p.codes_vec = (reinterpret_cast<uintptr_t>(p.q) & 7) == 0 && p.ldq % 8 == 0;
  if (norm) return vec ? launch_rows<T, true, true>(p, s) : launch_rows<T, true, false>(p, s);
  return vec ? launch_rows<T, false, true>(p, s) : launch_rows<T, false, false>(p, s);
}

cudaError_t launch_rows_any(const RowsParams& p, int dtype, bool norm, cudaStream_t s) {
  switch (dtype) {
    case PK_F16: return launch_rows_typed<__half>(p, norm, s);
    case PK_BF16: return launch_rows_typed<__nv_bfloat16>(p, norm, s);
    case PK_F32: return launch_rows_typed<float>(p, norm, s);
    default: return cudaErrorInvalidValue;
  }
}

template <typename T>
cudaError_t launch_dequantize_typed(const uint8_t* q, int64_t ldq, const float* scale, T* out,
                                    int64_t ldo, int64_t rows, int cols, int e4m3,
                                    cudaStream_t s) {
  const int items = (cols + 7) / 8 + 1;  // one more for the start of an unaligned row
  int tx = 32;
  while (tx < 256 && tx < items) tx *= 2;
  const int ty = 256 / tx;
  const int64_t gy = (rows + ty - 1) / ty;
  const dim3 grid(static_cast<unsigned>((items + tx - 1) / tx),
                  static_cast<unsigned>(gy < 65535 ? gy : 65535));
  const dim3 block(tx, ty);
  return launch_chained(dequantize_rows_kernel<T>, grid, block, s, q, ldq, scale, out, ldo, rows,
                        cols, e4m3);
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
