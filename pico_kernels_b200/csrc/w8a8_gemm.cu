// W8A8 products: out = (A8[M, K] @ W8[N, K]^T) * a_scale[m] * w_scale[n] (+ bias[n]),
// and their gated form act(gate) * up of two such products.
//
// Simple form: one 64 x 64 output tile per CTA, 4 x 4 outputs per thread, the
// operands staged 64 bytes of K at a time; int8 by four-way integer dot
// products into int32 (exact), e4m3 by fp32 multiply-adds.
#include <cuda_fp8.h>

#include "pk_common.cuh"

namespace pk {
namespace {

struct Params {
  const uint8_t* a;
  const uint8_t* w[2];
  const float* a_scale;
  const float* w_scale[2];
  const float* bias;
  void* out;
  int64_t lda, ldw[2], ldo;
  int64_t M;
  int N, K;
  int out_dtype, act;
};

constexpr int kTile = 64, kBK = 64;

__device__ __forceinline__ float gate(float g, int act) {
  // g * sigmoid(t): SiLU with t = g, GELU's tanh form with t = 2 sqrt(2/pi) (g + 0.044715 g^3)
  const float t = act == PK_ACT_SILU ? g : 1.5957691216057308f * (g + 0.044715f * g * g * g);
  return g / (1.0f + expf(-t));
}

__device__ __forceinline__ void store_out(void* out, int dtype, int64_t i, float v) {
  if (dtype == PK_F16)
    static_cast<__half*>(out)[i] = __float2half_rn(v);
  else
    store_elem(out, dtype, i, v);
}

template <bool kE4M3, bool kGated>
__global__ void __launch_bounds__(256) w8a8_kernel(const Params p) {
  constexpr int kW = kGated ? 2 : 1;
  __shared__ uint32_t sa[kTile][kBK / 4 + 1], sw[kW][kTile][kBK / 4 + 1];
  const int t = threadIdx.x, tx = t & 15, ty = t >> 4;
  const int64_t m0 = static_cast<int64_t>(blockIdx.y) * kTile;
  const int n0 = blockIdx.x * kTile;
  int acc_i[kW][4][4] = {};
  float acc_f[kW][4][4] = {};
  griddep_wait();
  griddep_launch_dependents();
  for (int k0 = 0; k0 < p.K; k0 += kBK) {
    for (int i = t; i < kTile * (kBK / 4); i += 256) {
      const int r = i / (kBK / 4), c = i % (kBK / 4);
      auto word = [&](const uint8_t* base, int64_t row, int64_t rows, int64_t ld) {
        uint32_t v = 0;
        for (int b = 0; b < 4; ++b)
          if (row < rows && k0 + 4 * c + b < p.K)
            v |= static_cast<uint32_t>(base[row * ld + k0 + 4 * c + b]) << (8 * b);
        return v;
      };
      sa[r][c] = word(p.a, m0 + r, p.M, p.lda);
      for (int w = 0; w < kW; ++w) sw[w][r][c] = word(p.w[w], n0 + r, p.N, p.ldw[w]);
    }
    __syncthreads();
    for (int c = 0; c < kBK / 4; ++c)
      for (int w = 0; w < kW; ++w)
        for (int i = 0; i < 4; ++i)
          for (int j = 0; j < 4; ++j) {
            const uint32_t x = sa[ty * 4 + i][c], y = sw[w][tx * 4 + j][c];
            if (kE4M3) {
              for (int b = 0; b < 4; ++b) {
                const auto f = [](uint32_t v) {
                  return __half2float(__half(__nv_cvt_fp8_to_halfraw(
                      static_cast<__nv_fp8_storage_t>(v & 0xff), __NV_E4M3)));
                };
                acc_f[w][i][j] = fmaf(f(x >> (8 * b)), f(y >> (8 * b)), acc_f[w][i][j]);
              }
            } else {
              acc_i[w][i][j] = __dp4a(static_cast<int>(x), static_cast<int>(y), acc_i[w][i][j]);
            }
          }
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int64_t m = m0 + ty * 4 + i;
      const int n = n0 + tx * 4 + j;
      if (m >= p.M || n >= p.N) continue;
      float v[kW];
      for (int w = 0; w < kW; ++w)
        v[w] = (kE4M3 ? acc_f[w][i][j] : static_cast<float>(acc_i[w][i][j])) * p.a_scale[m] *
               p.w_scale[w][n];
      float y = v[0];
      if (kGated)
        y = gate(v[0], p.act) * v[kW - 1];
      else if (p.bias != nullptr)
        y += p.bias[n];
      store_out(p.out, p.out_dtype, m * p.ldo + n, y);
    }
}

}  // namespace

cudaError_t launch_w8a8(const W8A8Args& g, cudaStream_t s, const char** why) {
  (void)why;
  Params p{};
  p.a = static_cast<const uint8_t*>(g.a);
  p.lda = g.lda;
  p.a_scale = g.a_scale;
  for (int i = 0; i < 2; ++i) {
    p.w[i] = static_cast<const uint8_t*>(g.w[i]);
    p.ldw[i] = g.ldw[i];
    p.w_scale[i] = g.w_scale[i];
  }
  p.bias = g.bias;
  p.out = g.out;
  p.ldo = g.ldo;
  p.M = g.M;
  p.N = static_cast<int>(g.N);
  p.K = static_cast<int>(g.K);
  p.out_dtype = g.out_dtype;
  p.act = g.act;
  const dim3 grid(static_cast<unsigned>((g.N + kTile - 1) / kTile),
                  static_cast<unsigned>((g.M + kTile - 1) / kTile));
  if (g.gated) {
    if (g.e4m3) w8a8_kernel<true, true><<<grid, 256, 0, s>>>(p);
    else w8a8_kernel<false, true><<<grid, 256, 0, s>>>(p);
  } else {
    if (g.e4m3) w8a8_kernel<true, false><<<grid, 256, 0, s>>>(p);
    else w8a8_kernel<false, false><<<grid, 256, 0, s>>>(p);
  }
  return cudaGetLastError();
}

}  // namespace pk
