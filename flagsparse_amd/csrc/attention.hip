// Attention over packed sequences, forward and backward.
#include "attn.hpp"

namespace fsp {
namespace {

constexpr int kTile = 64;

struct Tile {
  int first, rows, at, q_begin, nq, k_begin, nk, pad;
};

struct Shape {
  int heads, kv_heads, dim, causal, window;
  float scale;
};

// Query i of a sequence sees the keys [lo, hi).
__device__ __forceinline__ void seen_by(const Shape& s, const Tile& t, int i, int& lo, int& hi) {
  lo = 0;
  hi = t.nk;
  if (s.causal) {
    hi = i + t.nk - t.nq + 1;
    if (s.window && hi > s.window) lo = hi - s.window;
    if (hi < 0) hi = 0;
  }
}

// One wave a query row: 64 keys at a time, a lane to a key for the scores and to elements of the
// head for the products.
template <typename T>
__global__ __launch_bounds__(kWave) void attention_packed_kernel(
    Shape s, const Tile* __restrict__ tiles, const T* __restrict__ q, int64_t q_token,
    int64_t q_head, const T* __restrict__ k, int64_t k_token, int64_t k_head,
    const T* __restrict__ v, int64_t v_token, int64_t v_head, T* __restrict__ out,
    int64_t o_token, int64_t o_head, float* __restrict__ lse) {
  __shared__ float s_q[kAttnDimCap];
  const Tile t = tiles[blockIdx.x];
  const int a = blockIdx.y, lane = threadIdx.x, g = a / (s.heads / s.kv_heads);
  for (int r = 0; r < t.rows; ++r) {
    const int64_t row = t.first + r;
    const T* qr = q + row * q_token + a * q_head;
    __syncthreads();
    for (int d = lane; d < s.dim; d += kWave) s_q[d] = (float)qr[d];
    __syncthreads();
    int lo, hi;
    seen_by(s, t, t.at + r, lo, hi);
    float m = -INFINITY, l = 0, acc[2] = {0, 0};
    for (int j0 = lo; j0 < hi; j0 += kWave) {
      const int j = j0 + lane;
      float x = -INFINITY;
      if (j < hi) {
        const T* kr = k + (int64_t)(t.k_begin + j) * k_token + g * k_head;
        x = 0;
        for (int d = 0; d < s.dim; ++d) x += s_q[d] * (float)kr[d];
        x *= s.scale;
      }
      const float top = fmaxf(m, wave_max(x));
      const float base = top == -INFINITY ? 0.0f : top;
      const float p = expf(x - base), fade = expf(m - base);
      l = l * fade + wave_add(p);
      acc[0] *= fade;
      acc[1] *= fade;
      m = top;
      for (int e = 0; e < kWave && j0 + e < hi; ++e) {
        const float pe = __shfl(p, e);
        const T* vr = v + (int64_t)(t.k_begin + j0 + e) * v_token + g * v_head;
        for (int u = 0; u < 2; ++u)
          if (lane + u * kWave < s.dim) acc[u] += pe * (float)vr[lane + u * kWave];
      }
    }
    T* o = out + row * o_token + a * o_head;
    for (int u = 0; u < 2; ++u)
      if (lane + u * kWave < s.dim) o[lane + u * kWave] = (T)(l > 0 ? acc[u] / l : acc[u]);
    if (lane == 0) lse[row * s.heads + a] = m + logf(l);
  }
}

// Gradient of the queries, a wave a row as above; also writes delta = grad_out . out.
template <typename T>
__global__ __launch_bounds__(kWave) void attention_grad_q_kernel(
    Shape s, const Tile* __restrict__ tiles, const T* __restrict__ q, int64_t q_token,
    int64_t q_head, const T* __restrict__ k, int64_t k_token, int64_t k_head,
    const T* __restrict__ v, int64_t v_token, int64_t v_head, const T* __restrict__ out,
    int64_t o_token, int64_t o_head, const float* __restrict__ lse, const T* __restrict__ go,
    int64_t go_token, int64_t go_head, T* __restrict__ dq, int64_t dq_token, int64_t dq_head,
    float* __restrict__ delta) {
  __shared__ float s_q[kAttnDimCap], s_g[kAttnDimCap];
  const Tile t = tiles[blockIdx.x];
  const int a = blockIdx.y, lane = threadIdx.x, g = a / (s.heads / s.kv_heads);
  for (int r = 0; r < t.rows; ++r) {
    const int64_t row = t.first + r;
    __syncthreads();
    float dl = 0;
    for (int d = lane; d < s.dim; d += kWave) {
      s_q[d] = (float)q[row * q_token + a * q_head + d];
      s_g[d] = (float)go[row * go_token + a * go_head + d];
      dl += s_g[d] * (float)out[row * o_token + a * o_head + d];
    }
    __syncthreads();
    dl = wave_add(dl);
    if (lane == 0) delta[row * s.heads + a] = dl;
    const float e0 = lse[row * s.heads + a];
    int lo, hi;
    seen_by(s, t, t.at + r, lo, hi);
    float acc[2] = {0, 0};
    for (int j0 = lo; j0 < hi; j0 += kWave) {
      const int j = j0 + lane;
      float ds = 0;
      if (j < hi) {
        const T* kr = k + (int64_t)(t.k_begin + j) * k_token + g * k_head;
        const T* vr = v + (int64_t)(t.k_begin + j) * v_token + g * v_head;
        float x = 0, dp = 0;
        for (int d = 0; d < s.dim; ++d) {
          x += s_q[d] * (float)kr[d];
          dp += s_g[d] * (float)vr[d];
        }
        ds = expf(x * s.scale - e0) * (dp - dl) * s.scale;
      }
      for (int e = 0; e < kWave && j0 + e < hi; ++e) {
        const float de = __shfl(ds, e);
        const T* kr = k + (int64_t)(t.k_begin + j0 + e) * k_token + g * k_head;
        for (int u = 0; u < 2; ++u)
          if (lane + u * kWave < s.dim) acc[u] += de * (float)kr[lane + u * kWave];
      }
    }
    for (int u = 0; u < 2; ++u)
      if (lane + u * kWave < s.dim)
        dq[row * dq_token + a * dq_head + lane + u * kWave] = (T)acc[u];
  }
}

// Gradients of the keys and values, a wave a key row: 64 queries at a time.
template <typename T>
__global__ __launch_bounds__(kWave) void attention_grad_kv_kernel(
    Shape s, const Tile* __restrict__ tiles, const T* __restrict__ q, int64_t q_token,
    int64_t q_head, const T* __restrict__ k, int64_t k_token, int64_t k_head,
    const T* __restrict__ v, int64_t v_token, int64_t v_head, const float* __restrict__ lse,
    const T* __restrict__ go, int64_t go_token, int64_t go_head,
    const float* __restrict__ delta, T* __restrict__ dk, int64_t dk_token, int64_t dk_head,
    T* __restrict__ dv, int64_t dv_token, int64_t dv_head) {
  __shared__ float s_k[kAttnDimCap], s_v[kAttnDimCap];
  const Tile t = tiles[blockIdx.x];
  const int g = blockIdx.y, lane = threadIdx.x, group = s.heads / s.kv_heads;
  for (int r = 0; r < t.rows; ++r) {
    const int64_t row = t.first + r;
    const int j = t.at + r;
    __syncthreads();
    for (int d = lane; d < s.dim; d += kWave) {
      s_k[d] = (float)k[row * k_token + g * k_head + d];
      s_v[d] = (float)v[row * v_token + g * v_head + d];
    }
    __syncthreads();
    int lo = 0, hi = t.nq;  // the queries that see key j
    if (s.causal) {
      lo = j - t.nk + t.nq;
      if (s.window && lo < t.nq - s.window) hi = lo + s.window;
      if (lo < 0) lo = 0;
    }
    float ak[2] = {0, 0}, av[2] = {0, 0};
    for (int a = g * group; a < (g + 1) * group; ++a) {
      for (int i0 = lo; i0 < hi; i0 += kWave) {
        const int64_t i = t.q_begin + i0 + lane;
        float p = 0, ds = 0;
        if (i0 + lane < hi) {
          const T* qr = q + i * q_token + a * q_head;
          const T* gr = go + i * go_token + a * go_head;
          float x = 0, dp = 0;
          for (int d = 0; d < s.dim; ++d) {
            x += s_k[d] * (float)qr[d];
            dp += s_v[d] * (float)gr[d];
          }
          p = expf(x * s.scale - lse[i * s.heads + a]);
          ds = p * (dp - delta[i * s.heads + a]) * s.scale;
        }
        for (int e = 0; e < kWave && i0 + e < hi; ++e) {
          const float pe = __shfl(p, e), de = __shfl(ds, e);
          const T* qr = q + (int64_t)(t.q_begin + i0 + e) * q_token + a * q_head;
          const T* gr = go + (int64_t)(t.q_begin + i0 + e) * go_token + a * go_head;
          for (int u = 0; u < 2; ++u)
            if (lane + u * kWave < s.dim) {
              ak[u] += de * (float)qr[lane + u * kWave];
              av[u] += pe * (float)gr[lane + u * kWave];
            }
        }
      }
    }
    for (int u = 0; u < 2; ++u)
      if (lane + u * kWave < s.dim) {
        dk[row * dk_token + g * dk_head + lane + u * kWave] = (T)ak[u];
        dv[row * dv_token + g * dv_head + lane + u * kWave] = (T)av[u];
      }
  }
}

template <typename T>
const T* in(const void* p) { return static_cast<const T*>(p); }

Shape shape_of(const fsp_attention_packed_args& a) {
  return {(int)a.heads, (int)a.kv_heads, (int)a.dim, (int)a.causal, (int)a.window,
          (float)a.scale};
}

template <typename T>
int launch_forward(const fsp_attention_packed_args& a, hipStream_t st) {
  hipLaunchKernelGGL((attention_packed_kernel<T>), dim3((unsigned)a.n_q_tiles, (unsigned)a.heads),
                     dim3(kWave), 0, st, shape_of(a), reinterpret_cast<const Tile*>(a.q_tiles),
                     in<T>(a.q), a.q_token, a.q_head, in<T>(a.k), a.k_token, a.k_head, in<T>(a.v),
                     a.v_token, a.v_head, static_cast<T*>(a.out), a.out_token, a.out_head, a.lse);
  return check_hip(hipGetLastError(), "attention_packed_kernel launch");
}

template <typename T>
int launch_backward(const fsp_attention_packed_args& a, hipStream_t st) {
  if (a.n_q_tiles > 0) {
    hipLaunchKernelGGL((attention_grad_q_kernel<T>),
                       dim3((unsigned)a.n_q_tiles, (unsigned)a.heads), dim3(kWave), 0, st,
                       shape_of(a), reinterpret_cast<const Tile*>(a.q_tiles), in<T>(a.q),
                       a.q_token, a.q_head, in<T>(a.k), a.k_token, a.k_head, in<T>(a.v),
                       a.v_token, a.v_head, in<T>(a.out), a.out_token, a.out_head, a.lse,
                       in<T>(a.grad_out), a.grad_out_token, a.grad_out_head,
                       static_cast<T*>(a.grad_q), a.grad_q_token, a.grad_q_head,
                       static_cast<float*>(a.workspace));
    if (int rc = check_hip(hipGetLastError(), "attention_grad_q_kernel launch")) return rc;
  }
  if (a.n_k_tiles > 0) {
    hipLaunchKernelGGL((attention_grad_kv_kernel<T>),
                       dim3((unsigned)a.n_k_tiles, (unsigned)a.kv_heads), dim3(kWave), 0, st,
                       shape_of(a), reinterpret_cast<const Tile*>(a.k_tiles), in<T>(a.q),
                       a.q_token, a.q_head, in<T>(a.k), a.k_token, a.k_head, in<T>(a.v),
                       a.v_token, a.v_head, a.lse, in<T>(a.grad_out), a.grad_out_token,
                       a.grad_out_head, static_cast<const float*>(a.workspace),
                       static_cast<T*>(a.grad_k), a.grad_k_token, a.grad_k_head,
                       static_cast<T*>(a.grad_v), a.grad_v_token, a.grad_v_head);
    return check_hip(hipGetLastError(), "attention_grad_kv_kernel launch");
  }
  return FSP_OK;
}

int check_packed(const fsp_attention_packed_args& a, const std::string& who) {
  if (!attn_dtype(a.dtype)) return set_error(FSP_ENOTSUP, who + ": dtype");
  if (!attn_dim(a.dim)) return set_error(FSP_ENOTSUP, who + ": dim");
  if (a.kv_heads < 1 || a.heads < 1 || a.heads % a.kv_heads || a.heads > 0xffff)
    return set_error(FSP_EINVAL, who + ": heads must be a multiple of kv_heads");
  if (a.q_tokens < 0 || a.k_tokens < 0 || a.n_q_tiles < 0 || a.n_k_tiles < 0 || a.window < 0 ||
      a.q_tokens > 0x7fffffffLL || a.k_tokens > 0x7fffffffLL || a.window > 0x7fffffffLL ||
      a.n_q_tiles > kMaxBlocks / a.heads || a.n_k_tiles > kMaxBlocks / a.heads)
    return set_error(FSP_EINVAL, who + ": size out of range");
  if (a.window && !a.causal) return set_error(FSP_EINVAL, who + ": window needs causal");
  if ((a.n_q_tiles > 0 && (!a.q_tiles || !a.q || !a.out || !a.lse)) ||
      (a.n_k_tiles > 0 && !a.k_tiles) || (a.k_tokens > 0 && (!a.k || !a.v)))
    return set_error(FSP_EINVAL, who + ": null pointer");
  if (!aligned16(a.q, a.q_token, a.q_head) || !aligned16(a.k, a.k_token, a.k_head) ||
      !aligned16(a.v, a.v_token, a.v_head) || !aligned16(a.out, a.out_token, a.out_head))
    return set_error(FSP_EINVAL, who + ": rows must be 16-byte aligned");
  return FSP_OK;
}

}  // namespace
}  // namespace fsp

using namespace fsp;

extern "C" int64_t fsp_attention_packed_tile(void) { return kTile; }

extern "C" int fsp_attention_packed(const fsp_attention_packed_args* args, void* stream) {
  if (!args) return set_error(FSP_EINVAL, "fsp_attention_packed: null arguments");
  const fsp_attention_packed_args& a = *args;
  if (int rc = check_packed(a, "fsp_attention_packed")) return rc;
  if (a.n_q_tiles == 0) return FSP_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a.dtype == FSP_BF16 ? launch_forward<bf16>(a, st) : launch_forward<f16>(a, st);
}

extern "C" int fsp_attention_packed_backward(const fsp_attention_packed_args* args, void* stream) {
  if (!args) return set_error(FSP_EINVAL, "fsp_attention_packed_backward: null arguments");
  const fsp_attention_packed_args& a = *args;
  if (int rc = check_packed(a, "fsp_attention_packed_backward")) return rc;
  if ((a.n_q_tiles > 0 && (!a.grad_out || !a.grad_q || !a.workspace)) ||
      (a.n_k_tiles > 0 && (!a.grad_k || !a.grad_v)))
    return set_error(FSP_EINVAL, "fsp_attention_packed_backward: null pointer");
  if (!aligned16(a.grad_out, a.grad_out_token, a.grad_out_head) ||
      !aligned16(a.grad_q, a.grad_q_token, a.grad_q_head) ||
      !aligned16(a.grad_k, a.grad_k_token, a.grad_k_head) ||
      !aligned16(a.grad_v, a.grad_v_token, a.grad_v_head))
    return set_error(FSP_EINVAL, "fsp_attention_packed_backward: rows must be 16-byte aligned");
  hipStream_t st = static_cast<hipStream_t>(stream);
  return a.dtype == FSP_BF16 ? launch_backward<bf16>(a, st) : launch_backward<f16>(a, st);
}
