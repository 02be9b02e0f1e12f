// A Mamba layer for one token of each sequence: all that stands between its input and its output projection (gfx950).
//
//   u = silu(bias + conv weight . (tail, x))                 tail <- its last K - 1 inputs
//   (dt, B, C) = x_proj u,  delta = softplus(dt_proj dt + dt_bias)
//   h <- exp(delta A) h + delta u B,  out = (h C + Dp u) silu(z)
//
// Two launches. project_kernel forms u and its products with x_proj's columns, slice by slice of the channels; advance_kernel adds the
// slices' sums, forms delta and moves both states in place. Everything in between is float32.
#include "common.h"
#include "tsfast_hip.h"

using namespace tsf;

namespace {

constexpr int kThreads = 256;
constexpr int kCh = 64;     // channels of a step of a slice
constexpr int kRowsP = 16;  // rows (sequences) of a workgroup of project_kernel
constexpr int kRowsA = 4;   // and of advance_kernel, a wave each
constexpr int kMaxK = 8, kMaxN = 64;
constexpr int64_t kMaxP = 2048;  // R + 2 N

typedef float f32x4 __attribute__((ext_vector_type(4)));

struct StepArgs {
  const void *x, *z;
  void *tail, *out;
  float* h;
  const void *wc, *bc, *xp, *dp, *db;  // conv weight and bias, x_proj, dt_proj, dt_bias
  const float *A, *Dp;
  int64_t B, D, sx, sz, slice;  // slice: channels
  int N, R, P, slices, wc16, bc16, xp16, dp16, db16;
  float* part;  // [slices][B][P]
};

TSF_DEV float param(const void* p, int64_t i, int is_bf16) { return is_bf16 ? to_f32(((const bf16*)p)[i]) : ((const float*)p)[i]; }
// 8 values of a row at any alignment, the first n of them, zeros after
TSF_DEV void param8(float* v, const void* p, int64_t i, int n, int is_bf16) {
  if (n >= 8) {
    if (is_bf16) {
      uint32_t w[4];
      __builtin_memcpy(w, (const bf16*)p + i, 16);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[2 * k] = __uint_as_float(w[k] << 16), v[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
    } else {
      __builtin_memcpy(v, (const float*)p + i, 32);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? param(p, i + e, is_bf16) : 0.0f;
  }
}

// u of one channel of one row; `past` its K - 1 carried inputs, moved on by x where `move`
template <typename T, int K>
TSF_DEV float conv_step(const StepArgs& g, int64_t b, int64_t d, bool move) {
  T* tail = (T*)g.tail + (b * g.D + d) * (K - 1);
  T past[K];
#pragma unroll
  for (int k = 0; k < K - 1; ++k) past[k] = tail[k];
  past[K - 1] = ((const T*)g.x)[b * g.sx + d];
  float a = g.bc ? param(g.bc, d, g.bc16) : 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k) a = fmaf(param(g.wc, d * K + k, g.wc16), to_f32(past[k]), a);
  if (move) {
#pragma unroll
    for (int k = 0; k < K - 1; ++k) tail[k] = past[k + 1];
  }
  return a * sigmoid_fast(a);
}

// A workgroup: 16 rows, one slice of the channels, all of x_proj's P columns, 16 of them a wave at a time. The products are
// float32 matrix instructions; lane group lg has channels 8 lg .. of each 32.
template <typename T, int K>
__global__ void __launch_bounds__(kThreads) project_kernel(StepArgs g) {
  __shared__ float s_u[kRowsP][kCh + 4];
  const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, lg = lane >> 4, wave = tid >> 6;
  const int64_t slice = blockIdx.x % g.slices, b0 = blockIdx.x / g.slices * kRowsP;
  const int64_t c_end = (slice + 1) * g.slice < g.D ? (slice + 1) * g.slice : g.D;
  constexpr int kTiles = 2;  // of 16 columns that a wave has at once
  for (int p0 = wave * 16 * kTiles; p0 - wave * 16 * kTiles < g.P; p0 += 4 * 16 * kTiles) {
    f32x4 acc[kTiles];
#pragma unroll
    for (int i = 0; i < kTiles; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int64_t c = slice * g.slice; c < c_end; c += kCh) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kRowsP / 4; ++i) {
        const int r = wave + 4 * i;
        const int64_t b = b0 + r, d = c + lane;
        s_u[r][lane] = b < g.B && d < c_end ? conv_step<T, K>(g, b, d, false) : 0.0f;
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kCh; k += 32) {
        const int64_t d = c + k + 8 * lg;
        const int left = (int)(c_end - d < 8 ? (c_end > d ? c_end - d : 0) : 8);
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = s_u[li][k + 8 * lg + e];
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
          const int p = p0 + 16 * i + li;
          float w[8];
          param8(w, g.xp, (int64_t)(p < g.P ? p : 0) * g.D + d, p < g.P ? left : 0, g.xp16);
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[e], v[e], acc[i], 0, 0, 0);
        }
      }
    }
    // columns 4 lg + e of row li
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      const int p = p0 + 16 * i + 4 * lg;
      if (b0 + li < g.B) {
        float* to = g.part + (slice * g.B + b0 + li) * g.P + p;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (p + e < g.P) to[e] = acc[i][e];
      }
    }
  }
}

// A workgroup: 64 channels of up to 4 rows, a row a wave where it goes by channels. States: 4 lanes a channel, 4 states of each 16 a lane.
template <typename T, int K, int NV>
__global__ void __launch_bounds__(kThreads) advance_kernel(StepArgs g) {
  extern __shared__ float s_p[];  // [rows][P], then:
  __shared__ float4 s_c[kRowsA][kCh];  // delta, delta u, Dp u, silu(z)
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t tiles = (g.D + kCh - 1) / kCh, tile = blockIdx.x % tiles, b0 = blockIdx.x / tiles * kRowsA;
  const int rows = (int)(g.B - b0 < kRowsA ? g.B - b0 : kRowsA);
  const int N = g.N, R = g.R, P = g.P;

  // the states, on their way while the projections are formed
  const int q = tid & 3;
  const int64_t dh = tile * kCh + (tid >> 2);
  const bool act = dh < g.D;
  f32x4 h[kRowsA][NV];
#pragma unroll
  for (int r = 0; r < kRowsA; ++r)
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int n = 16 * j + 4 * q;
      const float* p = g.h + ((b0 + r) * g.D + dh) * N + n;
      h[r][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (act && r < rows) {
        if (n + 4 <= N) {
          __builtin_memcpy(&h[r][j], p, 16);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < N) h[r][j][e] = p[e];
        }
      }
    }
  f32x4 A2[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int n = 16 * j + 4 * q + e;
      A2[j][e] = act && n < N ? g.A[dh * N + n] * kLog2e : 0.0f;
    }

  for (int i = tid; i < rows * P; i += kThreads) {
    const float* p = g.part + b0 * P + i;
    float s = 0.0f;
    for (int k = 0; k < g.slices; ++k) s += p[k * g.B * P];
    s_p[i] = s;
  }
  __syncthreads();
  const int64_t d = tile * kCh + lane;
  if (wave < rows && d < g.D) {
    const int64_t b = b0 + wave;
    const float* dt = s_p + wave * P;
    float a = g.db ? param(g.db, d, g.db16) : 0.0f;
    for (int r = 0; r < R; r += 8) {
      float w[8];
      param8(w, g.dp, d * R + r, R - r, g.dp16);
#pragma unroll
      for (int e = 0; e < 8; ++e) a = fmaf(w[e], r + e < R ? dt[r + e] : 0.0f, a);
    }
    const float u = conv_step<T, K>(g, b, d, true), delta = softplus_fast(a), z = to_f32(((const T*)g.z)[b * g.sz + d]);
    s_c[wave][lane] = make_float4(delta, delta * u, g.Dp[d] * u, z * sigmoid_fast(z));
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRowsA; ++r) {
    if (r < rows) {
      const float4 c = s_c[r][tid >> 2];
      const float *Bt = s_p + r * P + R, *Ct = Bt + N;
      float y = 0.0f;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int n = 16 * j + 4 * q;
        if (n < N) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int m = n + e < N ? n + e : N - 1;
            h[r][j][e] = fmaf(fast_exp2(c.x * A2[j][e]), h[r][j][e], c.y * Bt[m]);
            y = fmaf(n + e < N ? h[r][j][e] : 0.0f, Ct[m], y);
          }
          if (act) {
            float* p = g.h + ((b0 + r) * g.D + dh) * N + n;
            if (n + 4 <= N) {
              __builtin_memcpy(p, &h[r][j], 16);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (n + e < N) p[e] = h[r][j][e];
            }
          }
        }
      }
      y += __shfl_xor(y, 1, kWave);
      y += __shfl_xor(y, 2, kWave);
      if (q == 0 && act) ((T*)g.out)[(b0 + r) * g.D + dh] = from_f32<T>((y + c.z) * c.w);
    }
  }
}

// ------------------------------------------------------------------------------------------ host
int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }
constexpr int64_t kMaxGrid = (1 << 24) - 1;

// Channels of a slice: 64, or more where the rows alone fill the chip
int64_t slice_for(int64_t B, int64_t D) {
  const int64_t wgs = up(B, kRowsP) * up(D, kCh), cus = device_cus();
  return up(wgs, 2 * cus) * kCh;
}

int step_status(int64_t B, int64_t D, int64_t N, int64_t R, int64_t K) {
  if (B < 0 || D < 0 || N < 1 || R < 1 || K < 2) return TSF_ERR_ARG;
  if (K > kMaxK || N > kMaxN || R + 2 * N > kMaxP || D > (int64_t)1 << 24 || B > (int64_t)1 << 31) return TSF_ERR_UNSUPPORTED;
  if (up(B, kRowsA) * up(D, kCh) > kMaxGrid) return TSF_ERR_UNSUPPORTED;
  return TSF_OK;
}

template <typename T, int K>
void launch_step(const StepArgs& a, hipStream_t st) {
  project_kernel<T, K><<<(unsigned)(up(a.B, kRowsP) * a.slices), kThreads, 0, st>>>(a);
  const unsigned grid = (unsigned)(up(a.B, kRowsA) * up(a.D, kCh));
  const size_t lds = (size_t)kRowsA * a.P * sizeof(float);
  if (a.N <= 16)
    advance_kernel<T, K, 1><<<grid, kThreads, lds, st>>>(a);
  else if (a.N <= 32)
    advance_kernel<T, K, 2><<<grid, kThreads, lds, st>>>(a);
  else
    advance_kernel<T, K, 4><<<grid, kThreads, lds, st>>>(a);
}
template <typename T>
void launch_k(const StepArgs& a, int64_t K, hipStream_t st) {
  switch (K) {
    case 2: launch_step<T, 2>(a, st); break;
    case 3: launch_step<T, 3>(a, st); break;
    case 4: launch_step<T, 4>(a, st); break;
    case 5: launch_step<T, 5>(a, st); break;
    case 6: launch_step<T, 6>(a, st); break;
    case 7: launch_step<T, 7>(a, st); break;
    default: launch_step<T, 8>(a, st); break;
  }
}

}  // namespace

extern "C" {

int64_t tsfast_hip_mamba_step_workspace_bytes(int64_t B, int64_t D, int64_t N, int64_t R, int64_t K) {
  if (step_status(B, D, N, R, K) != TSF_OK) return -1;
  if (B == 0 || D == 0) return 0;
  return up(D, slice_for(B, D)) * B * (R + 2 * N) * 4;
}

int tsfast_hip_mamba_step(int64_t B, int64_t D, int64_t N, int64_t R, int64_t K, int io_dtype, const int* param_dtypes, const void* x,
                          int64_t x_stride, const void* z, int64_t z_stride, void* conv_state, float* ssm_state, const void* conv_weight,
                          const void* conv_bias, const void* x_proj, const void* dt_proj, const void* dt_bias, const float* A,
                          const float* Dp, void* out, void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = step_status(B, D, N, R, K);
  if (rc != TSF_OK) return rc;
  if ((io_dtype != TSF_DTYPE_F32 && io_dtype != TSF_DTYPE_BF16) || !param_dtypes || x_stride < 0 || z_stride < 0) return TSF_ERR_ARG;
  if (B == 0 || D == 0) return TSF_OK;
  if (!x || !z || !conv_state || !ssm_state || !conv_weight || !x_proj || !dt_proj || !A || !Dp || !out) return TSF_ERR_ARG;
  if (!workspace || workspace_bytes < tsfast_hip_mamba_step_workspace_bytes(B, D, N, R, K)) return TSF_ERR_WORKSPACE;
  StepArgs a = {};
  a.x = x, a.z = z, a.tail = conv_state, a.out = out, a.h = ssm_state, a.wc = conv_weight, a.bc = conv_bias, a.xp = x_proj, a.dp = dt_proj;
  a.db = dt_bias, a.A = A, a.Dp = Dp, a.B = B, a.D = D, a.sx = x_stride, a.sz = z_stride, a.slice = slice_for(B, D);
  a.N = (int)N, a.R = (int)R, a.P = (int)(R + 2 * N), a.slices = (int)up(D, a.slice), a.part = (float*)workspace;
  int* const is16[5] = {&a.wc16, &a.bc16, &a.xp16, &a.dp16, &a.db16};
  for (int i = 0; i < 5; ++i) *is16[i] = param_dtypes[i] == TSF_DTYPE_BF16;
  if (io_dtype == TSF_DTYPE_BF16)
    launch_k<bf16>(a, K, (hipStream_t)stream);
  else
    launch_k<float>(a, K, (hipStream_t)stream);
  return tsf_launch_status();
}

}  // extern "C"
