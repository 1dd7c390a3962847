// Weight gradient of a linear layer from its input kept in 8 bits:
//   gW[o, k] = sum_t g[t, o] xh[t, k]
#include "checkpoint8.cuh"

namespace mhc {
namespace {

constexpr int kTile = 64, kDepth = 16;

// A 64 x 64 tile of gW a block, 4 x 4 values a thread, 16 tokens at a time
// through shared memory; the codes are expanded as they are staged.
template <typename TG, typename TW>
__global__ void __launch_bounds__(256)
    wgrad_plain_kernel(const TG* __restrict__ g, int64_t stride, const int8_t* __restrict__ codes,
                       const uint8_t* __restrict__ exps, TW* __restrict__ gw, int64_t T, int64_t O, int64_t K,
                       int64_t pitch) {
  __shared__ float sg[kDepth][kTile], sx[kDepth][kTile];
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int64_t o0 = (int64_t)blockIdx.y * kTile, k0 = (int64_t)blockIdx.x * kTile;
  float acc[4][4] = {};
  for (int64_t t0 = 0; t0 < T; t0 += kDepth) {
#pragma unroll
    for (int e = tid; e < kDepth * kTile; e += 256) {
      const int d = e / kTile, c = e % kTile;
      const int64_t t = t0 + d;
      sg[d][c] = t < T && o0 + c < O ? ck_f32(g[t * stride + o0 + c]) : 0.f;
      float v[1] = {0.f};
      if (t < T && k0 + c < K) ck_decode<1>(codes + t * pitch, exps + t * (pitch / kCkBlock), k0 + c, v);
      sx[d][c] = v[0];
    }
    __syncthreads();
#pragma unroll
    for (int d = 0; d < kDepth; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(sg[d][ty * 4 + i], sx[d][tx * 4 + j], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t o = o0 + ty * 4 + i, k = k0 + tx * 4 + j;
      if (o < O && k < K) ck_store(gw + o * K + k, acc[i][j]);
    }
}

template <typename TG, typename TW>
int launch_plain(const void* g, int64_t stride, const int8_t* codes, const uint8_t* exps, void* gw, int64_t T,
                 int64_t O, int64_t K, cudaStream_t st) {
  ProfScope p("checkpoint8_weight_grad", st);
  const dim3 grid((unsigned)((K + kTile - 1) / kTile), (unsigned)((O + kTile - 1) / kTile));
  wgrad_plain_kernel<TG, TW><<<grid, 256, 0, st>>>((const TG*)g, stride, codes, exps, (TW*)gw, T, O, K, ck_pitch(K));
  return check_launch("checkpoint8_weight_grad");
}

}  // namespace

int wgrad_device_error(int* value, bool) {
  *value = 0;  // nothing waits here
  return MHC_OK;
}

}  // namespace mhc

using namespace mhc;

extern "C" size_t mhc_checkpoint8_weight_grad_workspace_bytes(int64_t, int64_t, int64_t, int32_t, int32_t) {
  return 0;
}

extern "C" int mhc_checkpoint8_weight_grad(const void* grad_out, int32_t g_bf16, int64_t row_stride,
                                           const int8_t* codes, const uint8_t* exponents, void* grad_weight,
                                           int32_t gw_bf16, int64_t tokens, int64_t out_features,
                                           int64_t in_features, void*, size_t, void* stream) {
  const char* what = "checkpoint8_weight_grad";
  MHC_REQUIRE(tokens >= 0 && out_features >= 1 && in_features >= 1, MHC_ERR_INVALID_ARG,
              "%s: tokens must be >= 0, out_features and in_features >= 1 (got %lld, %lld, %lld)", what,
              (long long)tokens, (long long)out_features, (long long)in_features);
  MHC_REQUIRE(tokens < (1ll << 30) && out_features <= (1ll << 21) && in_features <= (1ll << 21), MHC_ERR_UNSUPPORTED,
              "%s: %lld tokens, %lld x %lld features are too many", what, (long long)tokens, (long long)out_features,
              (long long)in_features);
  MHC_REQUIRE_PTR(grad_weight);
  cudaStream_t st = (cudaStream_t)stream;
  if (tokens == 0) {
    cudaMemsetAsync(grad_weight, 0, (size_t)out_features * (size_t)in_features * (gw_bf16 ? 2 : 4), st);
    return check_launch(what);
  }
  MHC_REQUIRE_PTR(grad_out);
  MHC_REQUIRE(row_stride >= out_features || tokens == 1, MHC_ERR_INVALID_ARG, "%s: row_stride %lld < out_features %lld",
              what, (long long)row_stride, (long long)out_features);
  MHC_REQUIRE(codes != nullptr && exponents != nullptr, MHC_ERR_INVALID_ARG, "%s: codes and exponents must not be NULL",
              what);
  MHC_REQUIRE(aligned16(codes) && (reinterpret_cast<uintptr_t>(exponents) & 3) == 0, MHC_ERR_ALIGNMENT,
              "%s: codes must be 16-byte and exponents 4-byte aligned", what);
#define MHC_WGRAD(TG, TW) \
  launch_plain<TG, TW>(grad_out, row_stride, codes, exponents, grad_weight, tokens, out_features, in_features, st)
  return g_bf16 ? (gw_bf16 ? MHC_WGRAD(__nv_bfloat16, __nv_bfloat16) : MHC_WGRAD(__nv_bfloat16, float))
                : (gw_bf16 ? MHC_WGRAD(float, __nv_bfloat16) : MHC_WGRAD(float, float));
#undef MHC_WGRAD
}
