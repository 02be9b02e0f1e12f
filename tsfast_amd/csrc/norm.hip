// Norms before and after a block, fused with its gate and its residual scale (gfx950).
//
//   gated_norm     y = rms(x) w silu(gate), or rms(x silu(gate)) w, per group of a row's columns
//   residual_norm  new = r + scale rms(x) w_post,  y = rms(new) w
//
// with rms(x) = x / sqrt(mean(x^2) + eps). Every input is read once and every output written once: a row
// (of a group) stays in registers between its sums and its outputs, and the backward computes the
// normalised row again from the inputs it needs anyway, so the forward saves nothing. All arithmetic is fp32
// and each output is rounded once. HBM bounds them.
//
// A unit of TPU threads holds one row, in pieces of 16 bytes of x (8 bf16 or 4 fp32 columns) at any
// alignment, NIT pieces a thread; a workgroup walks rows and loads the next row's pieces before it works on
// this one's. Each thread keeps its columns' parameter gradients in registers over all its rows; they are summed
// over the workgroup's units, then over workgroups by reduce_kernel, in a fixed order.
#include <type_traits>

#include "common.h"
#include "tsfast_hip.h"

using namespace tsf;

namespace {

constexpr int kMaxWidth = 8192;
constexpr int kMaxGrid = (1 << 24) - 1;

// VL consecutive columns of a row
template <typename T, int VL>
struct Piece {
  T v[VL];
};
template <typename T, int VL>
TSF_DEV void load(Piece<T, VL>& p, const T* at, int n) {
  if (n >= VL) {
    __builtin_memcpy(&p, at, sizeof(p));
  } else {
#pragma unroll
    for (int e = 0; e < VL; ++e) {
      p.v[e] = from_f32<T>(0.0f);
      if (e < n) p.v[e] = at[e];
    }
  }
}
template <typename T, int VL>
TSF_DEV void store(T* at, const float* x, int n) {
  Piece<T, VL> p;
#pragma unroll
  for (int e = 0; e < VL; ++e) p.v[e] = from_f32<T>(x[e]);
  if (n >= VL) {
    __builtin_memcpy(at, &p, sizeof(p));
  } else {
#pragma unroll
    for (int e = 0; e < VL; ++e)
      if (e < n) at[e] = p.v[e];
  }
}

// The sums of K values over the TPU threads of a unit, in every thread.
template <int TPU, int K>
TSF_DEV void unit_sum(float (&v)[K]) {
#pragma unroll
  for (int m = (TPU < kWave ? TPU : kWave) / 2; m >= 1; m >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor(v[k], m, kWave);
  if constexpr (TPU > kWave) {
    __shared__ float part[K][TPU / kWave];
    const int wave = threadIdx.x / kWave;
    __syncthreads();  // the last sums have been read
    if (threadIdx.x % kWave == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) part[k][wave] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = 0.0f;
#pragma unroll
      for (int w = 0; w < TPU / kWave; ++w) v[k] += part[k][w];
    }
  }
}

constexpr int block_of(int tpu) { return tpu > 256 ? tpu : 256; }

// Adds up a workgroup's units' column sums and writes them to row blockIdx.x of `to` [blocks][columns].
template <int TPU, int NIT, int VL>
TSF_DEV void write_columns(const float (&acc)[NIT][VL], float* to, int width) {
  constexpr int U = block_of(TPU) / TPU;
  const int lane = threadIdx.x % TPU, unit = threadIdx.x / TPU;
  if constexpr (U == 1) {
#pragma unroll
    for (int i = 0; i < NIT; ++i)
#pragma unroll
      for (int e = 0; e < VL; ++e) {
        const int c = (i * TPU + lane) * VL + e;
        if (c < width) to[c] = acc[i][e];
      }
  } else {
    __shared__ float part[U][TPU * VL];
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < VL; ++e) part[unit][lane * VL + e] = acc[i][e];
      __syncthreads();
      for (int at = threadIdx.x; at < TPU * VL; at += block_of(TPU)) {
        float s = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u) s += part[u][at];
        const int c = i * TPU * VL + at;
        if (c < width) to[c] = s;
      }
    }
  }
}

struct Silu {
  float act, slope;
};
TSF_DEV Silu silu(float g) {
  const float s = 1.0f / (1.0f + __expf(-g));
  return {g * s, s * (1.0f + g * (1.0f - s))};
}

struct GatedArgs {
  const void *x, *gate, *dy;
  int64_t sx, sg, sdy, rows;
  const float* weight;
  void *y, *dx, *dgate;
  float* partial;  // [blockIdx.x][groups width]
  int groups, width, first;
  float eps;
};

template <typename T, int TPU, int NIT, bool BWD>
__global__ __launch_bounds__(block_of(TPU)) void gated_kernel(GatedArgs a) {
  constexpr int VL = 16 / sizeof(T), U = block_of(TPU) / TPU;
  const int lane = threadIdx.x % TPU, group = blockIdx.y;
  const int64_t col0 = (int64_t)group * a.width, wide = (int64_t)a.groups * a.width, step = (int64_t)gridDim.x * U;
  const T *x = (const T*)a.x + col0, *gate = (const T*)a.gate + col0, *dy = (const T*)a.dy + col0;
  int col[NIT];
  float w[NIT][VL];
#pragma unroll
  for (int i = 0; i < NIT; ++i) {
    col[i] = (i * TPU + lane) * VL;
#pragma unroll
    for (int e = 0; e < VL; ++e) w[i][e] = a.weight && col[i] + e < a.width ? a.weight[col0 + col[i] + e] : 1.0f;
  }
  Piece<T, VL> px[NIT], pg[NIT], pd[NIT];
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      const int n = row < a.rows ? a.width - col[i] : 0;
      load(px[i], x + row * a.sx + col[i], n);
      if (a.gate) load(pg[i], gate + row * a.sg + col[i], n);
      if (BWD) load(pd[i], dy + row * a.sdy + col[i], n);
    }
  };
  float dw[NIT][VL] = {};
  const float inv_n = 1.0f / (float)a.width;
  int64_t row = (int64_t)blockIdx.x * U + threadIdx.x / TPU;
  fetch(row);
  for (; row < a.rows; row += step) {
    float xs[NIT][VL], act[NIT][VL], slope[NIT][VL], d[NIT][VL];
#pragma unroll
    for (int i = 0; i < NIT; ++i)
#pragma unroll
      for (int e = 0; e < VL; ++e) {
        xs[i][e] = to_f32(px[i].v[e]);
        const Silu s = a.gate ? silu(to_f32(pg[i].v[e])) : Silu{1.0f, 0.0f};
        act[i][e] = s.act;
        if (BWD) {
          slope[i][e] = s.slope;
          d[i][e] = to_f32(pd[i].v[e]);
        }
      }
    fetch(row + step);
    // u: what is normalised; f: what multiplies it afterwards
    float sum[BWD ? 2 : 1] = {};
#pragma unroll
    for (int i = 0; i < NIT; ++i)
#pragma unroll
      for (int e = 0; e < VL; ++e) {
        const float u = a.first ? xs[i][e] * act[i][e] : xs[i][e];
        sum[0] = fmaf(u, u, sum[0]);
        if (BWD) sum[1] = fmaf(d[i][e] * w[i][e] * (a.first ? 1.0f : act[i][e]), u, sum[1]);
      }
    unit_sum<TPU>(sum);
    const float inv = rsqrtf(fmaf(sum[0], inv_n, a.eps));
    float mean = 0.0f;
    if constexpr (BWD) mean = sum[1] * inv * inv_n;
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      const int n = a.width - col[i];
      const int64_t at = row * wide + col0 + col[i];
      float o[VL], o2[VL];
#pragma unroll
      for (int e = 0; e < VL; ++e) {
        const float after = a.first ? 1.0f : act[i][e], norm = (a.first ? xs[i][e] * act[i][e] : xs[i][e]) * inv;
        if constexpr (!BWD) {
          o[e] = norm * w[i][e] * after;
        } else {
          dw[i][e] = fmaf(d[i][e] * after, norm, dw[i][e]);
          const float du = inv * (d[i][e] * w[i][e] * after - norm * mean);
          o[e] = a.first ? du * act[i][e] : du;
          o2[e] = slope[i][e] * (a.first ? du * xs[i][e] : d[i][e] * w[i][e] * norm);
        }
      }
      if (n > 0) {
        if constexpr (!BWD) {
          store<T, VL>((T*)a.y + at, o, n);
        } else {
          store<T, VL>((T*)a.dx + at, o, n);
          if (a.gate) store<T, VL>((T*)a.dgate + at, o2, n);
        }
      }
    }
  }
  if constexpr (BWD)
    if (a.weight) write_columns<TPU>(dw, a.partial + (int64_t)blockIdx.x * wide + col0, a.width);
}

struct ResidualArgs {
  const void *x, *res, *dnew, *dy;
  int64_t sx, sr, sdn, sdy, rows;
  const float *post, *scale, *weight;
  void *new_res, *y, *dx, *dres;
  float* partial;  // [2][blockIdx.x][width]: sum dy rms(new), sum dnew n1
  int width;
  float eps;
};

template <typename T, typename R, int TPU, int NIT, bool BWD>
__global__ __launch_bounds__(block_of(TPU)) void residual_kernel(ResidualArgs a) {
  constexpr int VL = 16 / sizeof(T), U = block_of(TPU) / TPU;
  const int lane = threadIdx.x % TPU;
  const int64_t step = (int64_t)gridDim.x * U;
  const T *x = (const T*)a.x, *dy = (const T*)a.dy;
  const R *res = (const R*)a.res, *dnew = (const R*)a.dnew;
  int col[NIT];
  float w[NIT][VL], sw[NIT][VL];  // sw: what the (normalised) branch is multiplied with
#pragma unroll
  for (int i = 0; i < NIT; ++i) {
    col[i] = (i * TPU + lane) * VL;
#pragma unroll
    for (int e = 0; e < VL; ++e) {
      const bool in = col[i] + e < a.width;
      w[i][e] = a.weight && in ? a.weight[col[i] + e] : 1.0f;
      sw[i][e] = (a.post && in ? a.post[col[i] + e] : 1.0f) * (a.scale && in ? a.scale[col[i] + e] : 1.0f);
    }
  }
  Piece<T, VL> px[NIT], pd[NIT];
  Piece<R, VL> pr[NIT], pn[NIT];
  auto fetch = [&](int64_t row) {
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      const int n = row < a.rows ? a.width - col[i] : 0;
      load(px[i], x + row * a.sx + col[i], n);
      load(pr[i], res + row * a.sr + col[i], n);
      if (BWD) {
        load(pd[i], dy + row * a.sdy + col[i], a.dy ? n : 0);
        load(pn[i], dnew + row * a.sdn + col[i], a.dnew ? n : 0);
      }
    }
  };
  float dw[NIT][VL] = {}, db[NIT][VL] = {};
  const float inv_n = 1.0f / (float)a.width;
  int64_t row = (int64_t)blockIdx.x * U + threadIdx.x / TPU;
  fetch(row);
  for (; row < a.rows; row += step) {
    float n1[NIT][VL], nw[NIT][VL], d[NIT][VL], dn[NIT][VL];
    float sum1[1] = {};
#pragma unroll
    for (int i = 0; i < NIT; ++i)
#pragma unroll
      for (int e = 0; e < VL; ++e) {
        n1[i][e] = to_f32(px[i].v[e]);
        nw[i][e] = to_f32(pr[i].v[e]);
        if (BWD) {
          d[i][e] = to_f32(pd[i].v[e]);
          dn[i][e] = to_f32(pn[i].v[e]);
        }
        sum1[0] = fmaf(n1[i][e], n1[i][e], sum1[0]);
      }
    fetch(row + step);
    float inv1 = 1.0f;
    if (a.post) {
      unit_sum<TPU>(sum1);
      inv1 = rsqrtf(fmaf(sum1[0], inv_n, a.eps));
    }
    float sum2[BWD ? 2 : 1] = {};
#pragma unroll
    for (int i = 0; i < NIT; ++i)
#pragma unroll
      for (int e = 0; e < VL; ++e) {
        n1[i][e] *= inv1;
        nw[i][e] = fmaf(n1[i][e], sw[i][e], nw[i][e]);
        sum2[0] = fmaf(nw[i][e], nw[i][e], sum2[0]);
        if (BWD) sum2[1] = fmaf(d[i][e] * w[i][e], nw[i][e], sum2[1]);
      }
    unit_sum<TPU>(sum2);
    const float inv2 = rsqrtf(fmaf(sum2[0], inv_n, a.eps));
    const int64_t at = row * a.width;
    if constexpr (!BWD) {
#pragma unroll
      for (int i = 0; i < NIT; ++i) {
        const int n = a.width - col[i];
        float o[VL];
#pragma unroll
        for (int e = 0; e < VL; ++e) o[e] = nw[i][e] * inv2 * w[i][e];
        if (n > 0) {
          store<R, VL>((R*)a.new_res + at + col[i], nw[i], n);
          store<T, VL>((T*)a.y + at + col[i], o, n);
        }
      }
    } else {
      const float mean2 = sum2[1] * inv2 * inv_n;
      float sum3[1] = {};
#pragma unroll
      for (int i = 0; i < NIT; ++i)
#pragma unroll
        for (int e = 0; e < VL; ++e) {
          const float n = nw[i][e] * inv2;
          dw[i][e] = fmaf(d[i][e], n, dw[i][e]);
          dn[i][e] += inv2 * (d[i][e] * w[i][e] - n * mean2);
          db[i][e] = fmaf(dn[i][e], n1[i][e], db[i][e]);
          sum3[0] = fmaf(dn[i][e] * sw[i][e], n1[i][e], sum3[0]);
        }
      float mean1 = 0.0f;
      if (a.post) {
        unit_sum<TPU>(sum3);
        mean1 = sum3[0] * inv_n;
      }
#pragma unroll
      for (int i = 0; i < NIT; ++i) {
        const int n = a.width - col[i];
        float o[VL];
#pragma unroll
        for (int e = 0; e < VL; ++e) o[e] = inv1 * (dn[i][e] * sw[i][e] - n1[i][e] * mean1);
        if (n > 0) {
          store<T, VL>((T*)a.dx + at + col[i], o, n);
          store<R, VL>((R*)a.dres + at + col[i], dn[i], n);
        }
      }
    }
  }
  if constexpr (BWD) {
    if (a.weight) write_columns<TPU>(dw, a.partial + (int64_t)blockIdx.x * a.width, a.width);
    if (a.post || a.scale) write_columns<TPU>(db, a.partial + ((int64_t)gridDim.x + blockIdx.x) * a.width, a.width);
  }
}

// Column sums of `in` [blocks][columns], each into up to two outputs with a factor a column (null: one).
constexpr int kRedCols = 64, kRedRows = 16;
__global__ __launch_bounds__(kRedCols* kRedRows) void reduce_kernel(const float* in, int blocks, int64_t columns, float* out1, const float* mul1,
                                                                    float* out2, const float* mul2) {
  __shared__ float part[kRedRows][kRedCols];
  const int lane = threadIdx.x % kRedCols, r = threadIdx.x / kRedCols;
  const int64_t c = (int64_t)blockIdx.x * kRedCols + lane;
  float s = 0.0f;
  if (c < columns)
#pragma unroll 8
    for (int b = r; b < blocks; b += kRedRows) s += in[(int64_t)b * columns + c];
  part[r][lane] = s;
  __syncthreads();
  if (r == 0 && c < columns) {
#pragma unroll
    for (int k = 1; k < kRedRows; ++k) s += part[k][lane];
    if (out1) out1[c] = mul1 ? s * mul1[c] : s;
    if (out2) out2[c] = mul2 ? s * mul2[c] : s;
  }
}

// ------------------------------------------------------------------------------------------ host

// Workgroups over rows: two on each CU, all groups together.
int64_t row_blocks(int64_t rows, int64_t groups) {
  int64_t n = (2 * (int64_t)device_cus() + groups - 1) / groups;
  if (n > rows) n = rows;
  return n < 1 ? 1 : n;
}

template <int N>
using Int = std::integral_constant<int, N>;

// The narrowest unit that holds a row in at most four pieces a thread.
template <typename F>
int by_width(int64_t pieces, F f) {
  if (pieces <= 16) return f(Int<16>{}, Int<1>{});
  if (pieces <= 32) return f(Int<16>{}, Int<2>{});
  if (pieces <= 64) return f(Int<64>{}, Int<1>{});
  if (pieces <= 128) return f(Int<64>{}, Int<2>{});
  if (pieces <= 192) return f(Int<64>{}, Int<3>{});
  if (pieces <= 256) return f(Int<64>{}, Int<4>{});
  if (pieces <= 512) return f(Int<256>{}, Int<2>{});
  if (pieces <= 1024) return f(Int<256>{}, Int<4>{});
  return f(Int<1024>{}, Int<2>{});
}

int norm_status(int64_t rows, int64_t groups, int64_t width, int dtype) {
  if (rows < 0 || groups < 1 || width < 1) return TSF_ERR_ARG;
  if (dtype != TSF_DTYPE_F32 && dtype != TSF_DTYPE_BF16) return TSF_ERR_ARG;
  if (width > kMaxWidth || groups > 65535 || groups * width > INT32_MAX || rows > ((int64_t)1 << 40)) return TSF_ERR_UNSUPPORTED;
  return TSF_OK;
}

template <typename T, bool BWD>
int gated(const GatedArgs& a, hipStream_t stream) {
  constexpr int VL = 16 / sizeof(T);
  const int64_t most = row_blocks(a.rows, a.groups);
  const int rc = by_width((a.width + VL - 1) / VL, [&](auto tpu, auto nit) {
    constexpr int TPU = decltype(tpu)::value, NIT = decltype(nit)::value, U = block_of(TPU) / TPU;
    const int64_t need = (a.rows + U - 1) / U;
    const int64_t blocks = BWD ? (need < most ? need : most) : (need < 4 * most ? need : 4 * most);
    gated_kernel<T, TPU, NIT, BWD><<<dim3((unsigned)blocks, (unsigned)a.groups), block_of(TPU), 0, stream>>>(a);
    return (int)blocks;
  });
  return rc;
}

template <typename T, typename R, bool BWD>
int residual(const ResidualArgs& a, hipStream_t stream) {
  constexpr int VL = 16 / sizeof(T);
  const int64_t most = row_blocks(a.rows, 1);
  return by_width((a.width + VL - 1) / VL, [&](auto tpu, auto nit) {
    constexpr int TPU = decltype(tpu)::value, NIT = decltype(nit)::value, U = block_of(TPU) / TPU;
    const int64_t need = (a.rows + U - 1) / U;
    const int64_t blocks = BWD ? (need < most ? need : most) : (need < 4 * most ? need : 4 * most);
    residual_kernel<T, R, TPU, NIT, BWD><<<(unsigned)blocks, block_of(TPU), 0, stream>>>(a);
    return (int)blocks;
  });
}

void reduce(const float* in, int blocks, int64_t columns, float* out1, const float* mul1, float* out2, const float* mul2, hipStream_t stream) {
  reduce_kernel<<<(unsigned)((columns + kRedCols - 1) / kRedCols), kRedCols * kRedRows, 0, stream>>>(in, blocks, columns, out1, mul1, out2, mul2);
}

void zero(float* p, int64_t n, hipStream_t stream) {
  if (p && n > 0) reduce(nullptr, 0, n, p, nullptr, nullptr, nullptr, stream);
}

}  // namespace

extern "C" {

int64_t tsfast_hip_norm_max_width(void) { return kMaxWidth; }

int64_t tsfast_hip_gated_norm_workspace_bytes(int64_t rows, int64_t groups, int64_t width) {
  if (norm_status(rows, groups, width, TSF_DTYPE_F32) != TSF_OK) return -1;
  return row_blocks(rows, groups) * groups * width * 4;
}

int64_t tsfast_hip_residual_norm_workspace_bytes(int64_t rows, int64_t width) {
  if (norm_status(rows, 1, width, TSF_DTYPE_F32) != TSF_OK) return -1;
  return 2 * row_blocks(rows, 1) * width * 4;
}

int tsfast_hip_gated_norm_fwd(int64_t rows, int64_t groups, int64_t width, int dtype, int gate_first, float eps, const void* x, int64_t x_stride,
                              const void* gate, int64_t gate_stride, const float* weight, void* y, void* stream) {
  const int rc = norm_status(rows, groups, width, dtype);
  if (rc != TSF_OK) return rc;
  if (rows == 0) return TSF_OK;
  if (!x || !y) return TSF_ERR_ARG;
  GatedArgs a = {};
  a.x = x, a.gate = gate, a.sx = x_stride, a.sg = gate_stride, a.rows = rows, a.weight = weight, a.y = y;
  a.groups = (int)groups, a.width = (int)width, a.first = gate_first && gate, a.eps = eps;
  (void)(dtype == TSF_DTYPE_BF16 ? gated<bf16, false>(a, (hipStream_t)stream) : gated<float, false>(a, (hipStream_t)stream));
  return tsf_launch_status();
}

int tsfast_hip_gated_norm_bwd(int64_t rows, int64_t groups, int64_t width, int dtype, int gate_first, float eps, const void* x, int64_t x_stride,
                              const void* gate, int64_t gate_stride, const float* weight, const void* grad_y, int64_t grad_y_stride, void* grad_x,
                              void* grad_gate, float* grad_weight, void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = norm_status(rows, groups, width, dtype);
  if (rc != TSF_OK) return rc;
  if (weight && !grad_weight) return TSF_ERR_ARG;
  const hipStream_t st = (hipStream_t)stream;
  if (rows == 0) {
    if (weight) zero(grad_weight, groups * width, st);
    return tsf_launch_status();
  }
  if (!x || !grad_y || !grad_x || (gate && !grad_gate)) return TSF_ERR_ARG;
  if (weight && (!workspace || workspace_bytes < tsfast_hip_gated_norm_workspace_bytes(rows, groups, width))) return TSF_ERR_WORKSPACE;
  GatedArgs a = {};
  a.x = x, a.gate = gate, a.dy = grad_y, a.sx = x_stride, a.sg = gate_stride, a.sdy = grad_y_stride, a.rows = rows, a.weight = weight;
  a.dx = grad_x, a.dgate = grad_gate, a.partial = (float*)workspace;
  a.groups = (int)groups, a.width = (int)width, a.first = gate_first && gate, a.eps = eps;
  const int blocks = dtype == TSF_DTYPE_BF16 ? gated<bf16, true>(a, st) : gated<float, true>(a, st);
  if (weight) reduce(a.partial, blocks, groups * width, grad_weight, nullptr, nullptr, nullptr, st);
  return tsf_launch_status();
}

int tsfast_hip_residual_norm_fwd(int64_t rows, int64_t width, int dtype, int res_dtype, float eps, const void* x, int64_t x_stride, const void* res,
                                 int64_t res_stride, const float* post_weight, const float* scale, const float* weight, void* new_residual, void* y,
                                 void* stream) {
  const int rc = norm_status(rows, 1, width, dtype);
  if (rc != TSF_OK) return rc;
  if (res_dtype != dtype && res_dtype != TSF_DTYPE_F32) return TSF_ERR_ARG;
  if (rows == 0) return TSF_OK;
  if (!x || !res || !new_residual || !y) return TSF_ERR_ARG;
  const hipStream_t st = (hipStream_t)stream;
  ResidualArgs a = {};
  a.x = x, a.res = res, a.sx = x_stride, a.sr = res_stride, a.rows = rows, a.post = post_weight, a.scale = scale, a.weight = weight;
  a.new_res = new_residual, a.y = y, a.width = (int)width, a.eps = eps;
  (void)(dtype == TSF_DTYPE_F32        ? residual<float, float, false>(a, st)
         : res_dtype == TSF_DTYPE_BF16 ? residual<bf16, bf16, false>(a, st)
                                       : residual<bf16, float, false>(a, st));
  return tsf_launch_status();
}

int tsfast_hip_residual_norm_bwd(int64_t rows, int64_t width, int dtype, int res_dtype, float eps, const void* x, int64_t x_stride, const void* res,
                                 int64_t res_stride, const float* post_weight, const float* scale, const float* weight, const void* grad_new,
                                 int64_t grad_new_stride, const void* grad_y, int64_t grad_y_stride, void* grad_x, void* grad_residual,
                                 float* grad_post_weight, float* grad_scale, float* grad_weight, void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = norm_status(rows, 1, width, dtype);
  if (rc != TSF_OK) return rc;
  if (res_dtype != dtype && res_dtype != TSF_DTYPE_F32) return TSF_ERR_ARG;
  if ((weight && !grad_weight) || (post_weight && !grad_post_weight) || (scale && !grad_scale)) return TSF_ERR_ARG;
  const hipStream_t st = (hipStream_t)stream;
  if (rows == 0) {
    if (weight) zero(grad_weight, width, st);
    if (post_weight) zero(grad_post_weight, width, st);
    if (scale) zero(grad_scale, width, st);
    return tsf_launch_status();
  }
  if (!x || !res || !grad_x || !grad_residual) return TSF_ERR_ARG;
  if (!workspace || workspace_bytes < tsfast_hip_residual_norm_workspace_bytes(rows, width)) return TSF_ERR_WORKSPACE;
  ResidualArgs a = {};
  a.x = x, a.res = res, a.dnew = grad_new, a.dy = grad_y, a.sx = x_stride, a.sr = res_stride, a.sdn = grad_new_stride, a.sdy = grad_y_stride;
  a.rows = rows, a.post = post_weight, a.scale = scale, a.weight = weight, a.dx = grad_x, a.dres = grad_residual, a.partial = (float*)workspace;
  a.width = (int)width, a.eps = eps;
  const int blocks = dtype == TSF_DTYPE_F32        ? residual<float, float, true>(a, st)
                     : res_dtype == TSF_DTYPE_BF16 ? residual<bf16, bf16, true>(a, st)
                                                   : residual<bf16, float, true>(a, st);
  if (weight) reduce(a.partial, blocks, width, grad_weight, nullptr, nullptr, nullptr, st);
  if (post_weight || scale)
    reduce(a.partial + (int64_t)blocks * width, blocks, width, post_weight ? grad_post_weight : nullptr, scale, scale ? grad_scale : nullptr, post_weight,
           st);
  return tsf_launch_status();
}

}  // extern "C"
