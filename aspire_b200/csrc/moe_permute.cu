// Tokens to their experts' rows and back, and the gradients.
//
//   dispatch:  rows[position[t, j]] = x[t];  rows past the last expert's are 0
//   combine:   y[t] = sum_j w[t, j] rows[position[t, j]]  (+ residual[t])
//   gradients: of dispatch: combine without weights; of combine:
//              d rows[position[t, j]] = w[t, j] dy[t],
//              d w[t, j] = <dy[t], rows[position[t, j]]>
//
// Bound by the bytes.  Every kernel goes by token: a block of 128 threads
// owns one, takes x[t] or dy[t] from memory once whatever top_k is (the combine's
// gradient goes over the row once for every four choices, the later times in the
// caches), and moves 16 bytes per thread and row; sums are in fp32 in the order of
// the choices, so nothing depends on which block runs first.  8192 tokens x 8 rows of 2048 bf16:
// dispatch 51 us and its gradient 46 us (91 % of the copy rate); 4099 x 4 rows
// of 4096: combine 29 us, its gradients 47 us.
#include "moe.cuh"

namespace aspire {

namespace {

template <typename T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int kN = 4;
  __device__ static __forceinline__ void unpack(const uint4& u, float* v) {
    v[0] = __uint_as_float(u.x);
    v[1] = __uint_as_float(u.y);
    v[2] = __uint_as_float(u.z);
    v[3] = __uint_as_float(u.w);
  }
  __device__ static __forceinline__ uint4 pack(const float* v) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int kN = 8;
  __device__ static __forceinline__ void unpack(const uint4& u, float* v) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  __device__ static __forceinline__ uint4 pack(const float* v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct Vec<__half> {
  static constexpr int kN = 8;
  __device__ static __forceinline__ void unpack(const uint4& u, float* v) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
  __device__ static __forceinline__ uint4 pack(const float* v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// The token's rows and weights, in shared memory: row -1 for no expert and
// for a position outside [0, tokens * top_k), which is reported.
__device__ __forceinline__ void load_slots(const MoePermuteParams& p, int64_t token, int32_t* row, float* weight) {
  const int j = threadIdx.x;
  if (j < p.top_k) {
    const int64_t slot = token * p.top_k + j;
    int32_t r = p.position[slot];
    if (r >= int64_t(p.tokens) * p.top_k) {
      record_status(p.status, ASPIRE_STATUS_BAD_ROW);
      r = -1;
    }
    row[j] = r;
    weight[j] = p.weights ? p.weights[slot] : 1.0f;
  }
  __syncthreads();
}

// Rows past the last expert's, shared among the blocks, become zero.
__device__ __forceinline__ void zero_tail(const MoePermuteParams& p, uint4* out, int64_t stride, int vecs) {
  const int64_t total = int64_t(p.tokens) * p.top_k;
  int64_t r = p.offsets[p.num_experts];
  r = r < 0 ? 0 : r;
  for (r += blockIdx.x; r < total; r += gridDim.x)
    for (int c = threadIdx.x; c < vecs; c += kMoeThreads) out[r * stride + c] = make_uint4(0, 0, 0, 0);
}

template <typename T>
__global__ void __launch_bounds__(kMoeThreads) aspire_moe_dispatch_kernel(MoePermuteParams p) {
  pdl_begin();
  constexpr int N = Vec<T>::kN;
  __shared__ int32_t row[kMoeMaxTopK];
  __shared__ float weight[kMoeMaxTopK];
  const int64_t token = blockIdx.x;
  const int vecs = p.width / N;
  const int64_t so = p.out_stride / N;
  const uint4* in = reinterpret_cast<const uint4*>(static_cast<const T*>(p.in) + token * p.in_stride);
  uint4* out = static_cast<uint4*>(p.out);
  load_slots(p, token, row, weight);
  for (int c = threadIdx.x; c < vecs; c += kMoeThreads) {
    const uint4 u = in[c];
    for (int j = 0; j < p.top_k; ++j)
      if (row[j] >= 0) out[row[j] * so + c] = u;
  }
  zero_tail(p, out, so, vecs);
}

template <typename T>
__global__ void __launch_bounds__(kMoeThreads) aspire_moe_combine_kernel(MoePermuteParams p) {
  pdl_begin();
  constexpr int N = Vec<T>::kN;
  __shared__ int32_t row[kMoeMaxTopK];
  __shared__ float weight[kMoeMaxTopK];
  const int64_t token = blockIdx.x;
  const int vecs = p.width / N;
  const int64_t si = p.in_stride / N;
  const uint4* in = static_cast<const uint4*>(p.in);
  uint4* out = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + token * p.out_stride);
  const uint4* res =
      p.residual ? reinterpret_cast<const uint4*>(static_cast<const T*>(p.residual) + token * p.residual_stride) : nullptr;
  load_slots(p, token, row, weight);
  for (int c = threadIdx.x; c < vecs; c += kMoeThreads) {
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
    for (int j0 = 0; j0 < p.top_k; j0 += 4) {
      uint4 u[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        u[j] = j0 + j < p.top_k && row[j0 + j] >= 0 ? in[row[j0 + j] * si + c] : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (j0 + j >= p.top_k || row[j0 + j] < 0) continue;
        float v[N];
        Vec<T>::unpack(u[j], v);
        const float w = weight[j0 + j];
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = fmaf(w, v[i], acc[i]);
      }
    }
    if (res) {
      float v[N];
      Vec<T>::unpack(res[c], v);
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] += v[i];
    }
    out[c] = Vec<T>::pack(acc);
  }
}

template <typename T>
__global__ void __launch_bounds__(kMoeThreads) aspire_moe_combine_grad_kernel(MoePermuteParams p) {
  pdl_begin();
  constexpr int N = Vec<T>::kN, J = 4;
  __shared__ int32_t row[kMoeMaxTopK];
  __shared__ float weight[kMoeMaxTopK];
  __shared__ float part[J][kMoeThreads / 32];
  const int64_t token = blockIdx.x;
  const int vecs = p.width / N;
  const int64_t si = p.in_stride / N, so = p.out_stride / N;
  const uint4* in = static_cast<const uint4*>(p.in);
  uint4* out = static_cast<uint4*>(p.out);
  const uint4* grad = reinterpret_cast<const uint4*>(static_cast<const T*>(p.grad) + token * p.grad_stride);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  load_slots(p, token, row, weight);
  for (int j0 = 0; j0 < p.top_k; j0 += J) {
    float dot[J];
#pragma unroll
    for (int j = 0; j < J; ++j) dot[j] = 0.f;
    for (int c = threadIdx.x; c < vecs; c += kMoeThreads) {
      float g[N];
      Vec<T>::unpack(grad[c], g);
      uint4 u[J];
#pragma unroll
      for (int j = 0; j < J; ++j)
        u[j] = p.grad_weights && j0 + j < p.top_k && row[j0 + j] >= 0 ? in[row[j0 + j] * si + c]
                                                                      : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        if (j0 + j >= p.top_k || row[j0 + j] < 0) continue;
        float v[N];
        Vec<T>::unpack(u[j], v);
#pragma unroll
        for (int i = 0; i < N; ++i) dot[j] = fmaf(g[i], v[i], dot[j]);
        if (out) {
          const float w = weight[j0 + j];
#pragma unroll
          for (int i = 0; i < N; ++i) v[i] = w * g[i];
          out[row[j0 + j] * so + c] = Vec<T>::pack(v);
        }
      }
    }
    if (p.grad_weights) {
#pragma unroll
      for (int j = 0; j < J; ++j) {
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) dot[j] += __shfl_xor_sync(0xffffffffu, dot[j], d);
        if (lane == 0) part[j][warp] = dot[j];
      }
      __syncthreads();
      if (threadIdx.x < J && j0 + int(threadIdx.x) < p.top_k) {
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < kMoeThreads / 32; ++w) s += part[threadIdx.x][w];
        p.grad_weights[token * p.top_k + j0 + threadIdx.x] = s;
      }
      __syncthreads();
    }
  }
  if (out) zero_tail(p, out, so, vecs);
}

}  // namespace

MoePermuteKernel moe_dispatch_kernel(int32_t type) {
  if (type == ASPIRE_T_F32) return aspire_moe_dispatch_kernel<float>;
  if (type == ASPIRE_T_BF16) return aspire_moe_dispatch_kernel<__nv_bfloat16>;
  return aspire_moe_dispatch_kernel<__half>;
}
MoePermuteKernel moe_combine_kernel(int32_t type) {
  if (type == ASPIRE_T_F32) return aspire_moe_combine_kernel<float>;
  if (type == ASPIRE_T_BF16) return aspire_moe_combine_kernel<__nv_bfloat16>;
  return aspire_moe_combine_kernel<__half>;
}
MoePermuteKernel moe_combine_grad_kernel(int32_t type) {
  if (type == ASPIRE_T_F32) return aspire_moe_combine_grad_kernel<float>;
  if (type == ASPIRE_T_BF16) return aspire_moe_combine_grad_kernel<__nv_bfloat16>;
  return aspire_moe_combine_grad_kernel<__half>;
}

}  // namespace aspire
