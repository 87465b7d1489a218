// Attention over packed sequences, forward and backward.
#include "attn.hpp"

namespace fsp {
namespace {

constexpr int kTile = 128;  // query rows of a workgroup, 32 a wave

constexpr int64_t kTokenStep = 1 << 23;  // 64 rows' bytes are a 32-bit offset

struct Tile {
  int first, rows, at, q_begin, nq, k_begin, nk, pad;
};

struct Shape {
  int heads, kv_heads, dim, causal, window;
  float scale;
};

// Workgroups go to the 8 XCDs in turn.  Where the heads divide by them, each XCD has heads of its own, so
// that the tiles it works on at a time read the same keys through its L2; within an XCD (and
// otherwise over all of them) the tiles run in the list's order, heavy ones first.
__device__ __forceinline__ void tile_and_head(int block, int n_tiles, int heads, int& tile, int& head) {
  if (heads % 8 == 0) {
    const int per = heads / 8, j = block >> 3;
    tile = j / per;
    head = (block & 7) * per + j % per;
  } else {
    tile = block / heads;
    head = block % heads;
  }
}

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

// Keys of one step, and how their rows lie in LDS: PITCH bytes each in chunks of 16, the chunks of a
// row permuted so that the lanes of one read meet different banks (K: by the row, for reads of one
// chunk of many rows; V: by the row's place in four, for transposed reads of four rows).
constexpr int kKeys = 64;

template <int DP>
struct Lay {
  static constexpr int PITCH = DP <= 64 ? 128 : 256;
  static constexpr int CH = PITCH / 16;
  static constexpr int BYTES = kKeys * PITCH;
  __device__ static int swizzle_k(int row) { return row & (CH - 1); }
  __device__ static int swizzle_v(int row) { return CH == 8 ? (row & 2) << 1 : (row & 3) << 2; }
};

// Rows [0, n) of a 16-bit array, ``bytes`` apart, straight to LDS: 1024 bytes a wave and load.  What lies
// past the rows or the head's dim is read as zero: the buffer's bounds end there.
template <int DP, bool V>
__device__ __forceinline__ void load_rows(char* lds, const void* src, int n, uint32_t bytes, int dim,
                                          int wave, int lane) {
  typedef Lay<DP> L;
  const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<void*>(src), 0, (int)((uint32_t)(n - 1) * bytes + 2 * dim), 0x00027000);
  constexpr int PER = L::BYTES / 1024 / 4;  // loads of a wave
  constexpr int ROWS = 1024 / L::PITCH;     // rows of a load
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int row = (wave * PER + i) * ROWS + lane / L::CH;
    const int chunk = (lane % L::CH) ^ (V ? L::swizzle_v(row) : L::swizzle_k(row));
    const uint32_t at = 8 * chunk < dim ? row * bytes + 16 * chunk : 0x80000000u;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        rsrc, (__attribute__((address_space(3))) void*)(lds + (wave * PER + i) * 1024), 16, (int)at,
        0, 0, 0);
  }
}

template <typename T>
__device__ __forceinline__ V8<T> to16(const f32x16& x, int at) {
  f32x8 v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = x[at + e];
  return __builtin_convertvector(v, V8<T>);
}

// Scores are scale * q . k, and weights exp(score - max) = exp2(c q . k - c max) with c = scale *
// log2(e) > 0: a negative scale turns q's sign, a zero one makes q zero.
template <typename T>
__device__ __forceinline__ V8<T> scaled_sign(V8<T> q, float scale) {
  if (scale > 0) return q;
  return scale < 0 ? -q : V8<T>{};
}

template <typename T, int DP>
__global__ __launch_bounds__(256, 2) void attention_packed_kernel(
    Shape s, const Tile* __restrict__ tiles, int n_tiles, const T* __restrict__ q, int64_t q_token,
    int64_t q_head, const T* __restrict__ k, int64_t k_token, int64_t k_head,
    const T* __restrict__ v, int64_t v_token, int64_t v_head, T* __restrict__ out,
    int64_t o_token, int64_t o_head, float* __restrict__ lse) {
  typedef Lay<DP> L;
  constexpr int NS = DP / 16, NT = DP / 32;
  __shared__ __attribute__((aligned(1024))) char s_k0[L::BYTES], s_v0[L::BYTES], s_k1[L::BYTES],
      s_v1[L::BYTES];
  int tile, a;
  tile_and_head(blockIdx.x, n_tiles, s.heads, tile, a);
  const Tile t = tiles[tile];
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = a / (s.heads / s.kv_heads);
  const int mine = wave * 32 + col;  // this lane's row of the tile
  const bool active = wave * 32 < t.rows;

  V8<T> qf[NS];
  {
    const T* qr = q + (t.first + (int64_t)min(mine, t.rows - 1)) * q_token + a * q_head;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
      const int d = 16 * i + 8 * half;
      const V8<T> x = *reinterpret_cast<const V8<T>*>(qr + (d < s.dim ? d : 0));
      qf[i] = d < s.dim ? scaled_sign<T>(x, s.scale) : V8<T>{};
    }
  }
  const float c = s.scale == 0 ? 1.0f : fabsf(s.scale) * kLog2e;

  // the keys that this lane's row sees, and those of the wave's first and last rows
  int lo, hi, lo0, hi0, lo1, hi1, lot, hit, none;
  seen_by(s, t, t.at + min(mine, t.rows - 1), lo, hi);
  seen_by(s, t, t.at + min(wave * 32, t.rows - 1), lo0, hi0);
  seen_by(s, t, t.at + min(wave * 32 + 31, t.rows - 1), lo1, hi1);
  seen_by(s, t, t.at, lot, none);
  seen_by(s, t, t.at + t.rows - 1, none, hit);

  f32x16 o[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) o[i] = f32x16{};
  float top = -INFINITY, sum = 0;

  const T* kb = k + (int64_t)t.k_begin * k_token + g * k_head;
  const T* vb = v + (int64_t)t.k_begin * v_token + g * v_head;
  auto load = [&](int j0, char* sk, char* sv) {
    const int n = min(kKeys, t.nk - j0);
    load_rows<DP, false>(sk, kb + j0 * k_token, n, (uint32_t)(2 * k_token), s.dim, wave, lane);
    load_rows<DP, true>(sv, vb + j0 * v_token, n, (uint32_t)(2 * v_token), s.dim, wave, lane);
  };
  const int k_at = col * L::PITCH + ((half ^ (col & (L::CH - 1))) << 4);
  int v_at[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const int j = lane & 15, row = 4 * half + (j >> 2);
    const int chunk = (4 * i + 2 * ((lane >> 4) & 1) + ((j & 3) >> 1)) ^ L::swizzle_v(row);
    v_at[i] = row * L::PITCH + chunk * 16 + (j & 1) * 8;
  }

  auto step = [&](int j0, const char* sk_, const char* sv_) {
    if (!active || j0 >= hi1 || j0 + kKeys <= lo0) return;
    const lds_char* sk = (const lds_char*)sk_;
    const lds_char* sv = (const lds_char*)sv_;
    f32x16 x[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      x[u] = f32x16{};
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const V8<T> kf = __builtin_bit_cast(
            V8<T>, *(const lds_s16x8*)(sk + (k_at ^ (i * 32)) + u * 32 * L::PITCH));
        x[u] = mfma32(kf, qf[i], x[u]);
      }
    }
    if (j0 + kKeys > hi0 || j0 < lo1) {
      const int first = lo - j0 - 4 * half, last = hi - j0 - 4 * half;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int j = 32 * u + 8 * (r / 4) + r % 4;
          x[u][r] = j >= first && j < last ? x[u][r] : -INFINITY;
        }
    }
    float m = x[0][0];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) m = fmaxf(m, x[u][r]);
    m = fmaxf(m, other_half(m));
    // The weights are taken against an older maximum until a row's grows by more than 2^8 of it
    if (__any((m - top) * c > 8.0f)) {
      const float now = fmaxf(top, m);
      const float fade = top == -INFINITY ? 0.0f : exp2f((top - now) * c);
      top = now;
      sum *= fade;
#pragma unroll
      for (int i = 0; i < NT; ++i) o[i] *= fade;
    }
    const float base = top == -INFINITY ? 0.0f : top * c;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        x[u][r] = __builtin_amdgcn_exp2f(fmaf(x[u][r], c, -base));
        sum += x[u][r];
      }
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // 16 keys: the ones that this lane holds the weights of
      const V8<T> pf = to16<T>(x[i / 2], 8 * (i % 2));
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const s16x4 low = lds_transposed(sv + v_at[n] + 16 * i * L::PITCH);
        const s16x4 high = lds_transposed(sv + v_at[n] + (16 * i + 8) * L::PITCH);
        const V8<T> vf = __builtin_bit_cast(
            V8<T>, __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7));
        o[n] = mfma32(vf, pf, o[n]);
      }
    }
  };

  int j0 = lot;
  if (j0 < hit) load(j0, s_k0, s_v0);
  __syncthreads();
  while (j0 < hit) {
    if (j0 + kKeys < hit) load(j0 + kKeys, s_k1, s_v1);
    step(j0, s_k0, s_v0);
    __syncthreads();
    j0 += kKeys;
    if (j0 >= hit) break;
    if (j0 + kKeys < hit) load(j0 + kKeys, s_k0, s_v0);
    step(j0, s_k1, s_v1);
    __syncthreads();
    j0 += kKeys;
  }

  sum += other_half(sum);
  if (mine >= t.rows) return;
  const int64_t row = t.first + mine;
  const float inv = sum > 0 ? 1.0f / sum : (sum == 0 ? 0.0f : sum);
  if (half == 0) lse[row * s.heads + a] = sum == 0 ? -INFINITY : (top * c + log2f(sum)) * kLn2;
  T* to = out + row * o_token + a * o_head;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const int d = 32 * i + 2 * r + 4 * half;
      if (d < s.dim) {
        f32x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = sum == 0 ? 0.0f : o[i][r + e] * inv;
        *reinterpret_cast<V4<T>*>(to + d) = __builtin_convertvector(y, V4<T>);
      }
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

template <typename T, int DP>
int launch_forward(const fsp_attention_packed_args& a, hipStream_t st) {
  hipLaunchKernelGGL((attention_packed_kernel<T, DP>), dim3((unsigned)(a.n_q_tiles * a.heads)),
                     dim3(256), 0, st, shape_of(a), reinterpret_cast<const Tile*>(a.q_tiles),
                     (int)a.n_q_tiles, in<T>(a.q), a.q_token, a.q_head, in<T>(a.k), a.k_token,
                     a.k_head, in<T>(a.v), a.v_token, a.v_head, static_cast<T*>(a.out),
                     a.out_token, a.out_head, a.lse);
  return check_hip(hipGetLastError(), "attention_packed_kernel launch");
}

template <typename T>
int launch_forward_dim(const fsp_attention_packed_args& a, hipStream_t st) {
  if (a.dim <= 64) return launch_forward<T, 64>(a, st);
  if (a.dim <= 96) return launch_forward<T, 96>(a, st);
  return launch_forward<T, 128>(a, st);
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
  if ((a.k_tokens > 1 && (a.k_token < a.dim || a.v_token < a.dim)) || a.k_token > kTokenStep ||
      a.v_token > kTokenStep)
    return set_error(FSP_EINVAL, who + ": a key's step must lie between dim and 2^23");
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
  return a.dtype == FSP_BF16 ? launch_forward_dim<bf16>(a, st) : launch_forward_dim<f16>(a, st);
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
