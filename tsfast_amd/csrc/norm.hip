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
// A unit of TPU threads holds one row (of a group), in pieces of 16 bytes of x (8 bf16 or 4 fp32 columns) at any
// alignment, NIT pieces a thread; it walks rows and loads the next row's pieces before it works on this one's. Each
// thread keeps its columns' parameter gradients in registers over all its rows; reduce_kernel sums them over the
// units in a fixed order.
#include <type_traits>

#include "common.h"
#include "tsfast_hip.h"

using namespace tsf;

namespace {

constexpr int kMaxWidth = 8192;

// VL consecutive columns of a row as they lie in memory, the first n of them, zeros after. Words, not columns: a loaded piece
// must not be taken apart before it is used, or the wait for it comes right after the load.
template <typename T, int VL>
struct Piece {
  uint32_t w[VL * sizeof(T) / 4];
};
template <typename T, int VL>
TSF_DEV void load(Piece<T, VL>& p, const T* at, int n) {
  if (n >= VL) {
    __builtin_memcpy(&p, at, sizeof(p));
  } else {
#pragma unroll
    for (int k = 0; k < (int)(sizeof(p) / 4); ++k) {
      if constexpr (sizeof(T) == 2) {
        const uint32_t low = 2 * k < n ? (uint32_t)at[2 * k].bits : 0u, high = 2 * k + 1 < n ? (uint32_t)at[2 * k + 1].bits : 0u;
        p.w[k] = low | high << 16;
      } else {
        p.w[k] = k < n ? __float_as_uint(at[k]) : 0u;
      }
    }
  }
}
template <typename T, int VL>
TSF_DEV float value(const Piece<T, VL>& p, int e) {
  if constexpr (sizeof(T) == 2) return __uint_as_float(e & 1 ? p.w[e / 2] & 0xffff0000u : p.w[e / 2] << 16);
  return __uint_as_float(p.w[e]);
}
template <typename T, int VL>
TSF_DEV void store(T* at, const float* x, int n) {
  T v[VL];
#pragma unroll
  for (int e = 0; e < VL; ++e) v[e] = from_f32<T>(x[e]);
  if (n >= VL) {
    __builtin_memcpy(at, v, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < VL; ++e)
      if (e < n) at[e] = v[e];
  }
}

constexpr int block_of(int tpu) { return tpu > kWave ? tpu : 256; }

// The sums of K values over the TPU threads of a unit, in every thread. Units of several waves take turns with two
// places in LDS, so that one barrier a sum is enough: nobody writes a place before all have read its last sums.
template <int TPU, int K>
TSF_DEV void unit_sum(float (&v)[K], int& turn) {
#pragma unroll
  for (int m = (TPU < kWave ? TPU : kWave) / 2; m >= 1; m >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor(v[k], m, kWave);
  if constexpr (TPU > kWave) {
    constexpr int W = TPU / kWave;
    __shared__ float part[2][2][W];
    if (threadIdx.x % kWave == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) part[turn][k][threadIdx.x / kWave] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = 0.0f;
#pragma unroll
      for (int w = 0; w < W; ++w) v[k] += part[turn][k][w];
    }
    turn ^= 1;
  }
}

// A unit's column sums to its own row of `to`.
template <int TPU, int NIT, int VL>
TSF_DEV void write_columns(const float (&acc)[NIT][VL], float* to, int width) {
  const int lane = threadIdx.x % TPU;
#pragma unroll
  for (int i = 0; i < NIT; ++i) store<float, VL>(to + (i * TPU + lane) * VL, acc[i], width - (i * TPU + lane) * VL);
}

// A parameter's values of a thread's columns; one where there is none.
template <int VL>
TSF_DEV void load_param(float (&w)[VL], const float* p, int n) {
  if (p && n >= VL) {
    __builtin_memcpy(w, p, sizeof(w));
  } else {
#pragma unroll
    for (int e = 0; e < VL; ++e) w[e] = p && e < n ? p[e] : 1.0f;
  }
}

struct Silu {
  float act, slope;
};
TSF_DEV Silu silu(float g) {
  const float s = sigmoid_fast(g);
  return {g * s, s * (1.0f + g * (1.0f - s))};
}

struct GatedArgs {
  const void *x, *gate, *dy;
  int64_t sx, sg, sdy, rows;
  const float* weight;
  void *y, *dx, *dgate;
  float* partial;  // [unit][width], which is [unit / groups][groups width]
  int groups, width, first;
  float eps;
};

template <typename T, int TPU, int NIT, bool BWD>
__global__ __launch_bounds__(block_of(TPU)) void gated_kernel(GatedArgs a) {
  constexpr int VL = 16 / sizeof(T), U = block_of(TPU) / TPU;
  // units go through the groups of a row and then the rows; their number in a launch is a multiple of the groups, so that
  // a unit stays with its group's columns
  const int lane = threadIdx.x % TPU, slot = blockIdx.x * U + threadIdx.x / TPU, group = slot % a.groups;
  const int64_t col0 = (int64_t)group * a.width, wide = (int64_t)a.groups * a.width, step = gridDim.x * U / a.groups;
  const T *x = (const T*)a.x + col0, *gate = (const T*)a.gate + col0, *dy = (const T*)a.dy + col0;
  int col[NIT], turn = 0;
  float w[NIT][VL];
#pragma unroll
  for (int i = 0; i < NIT; ++i) {
    col[i] = (i * TPU + lane) * VL;
    load_param(w[i], a.weight ? a.weight + col0 + col[i] : nullptr, a.width - col[i]);
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
  int64_t row = slot / a.groups;
  fetch(row);
  for (; row < a.rows; row += step) {
    float xs[NIT][VL], act[NIT][VL], slope[NIT][VL], d[NIT][VL];
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
#pragma unroll
      for (int e = 0; e < VL; ++e) {
        xs[i][e] = value(px[i], e);
        const Silu s = a.gate ? silu(value(pg[i], e)) : Silu{1.0f, 0.0f};
        act[i][e] = s.act;
        if (BWD) {
          slope[i][e] = s.slope;
          d[i][e] = value(pd[i], e);
        }
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
    unit_sum<TPU>(sum, turn);
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
    if (a.weight) write_columns<TPU>(dw, a.partial + (int64_t)slot * a.width, a.width);
}

struct ResidualArgs {
  const void *x, *res, *dnew, *dy;
  int64_t sx, sr, sdn, sdy, rows;
  const float *post, *scale, *weight;
  void *new_res, *y, *dx, *dres;
  float* partial;  // [2][unit][width]: sum dy rms(new), sum dnew n1
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
  int col[NIT], turn = 0;
  float w[NIT][VL], sw[NIT][VL];  // sw: what the (normalised) branch is multiplied with
#pragma unroll
  for (int i = 0; i < NIT; ++i) {
    col[i] = (i * TPU + lane) * VL;
    const int n = a.width - col[i];
    float scale[VL];
    load_param(w[i], a.weight ? a.weight + col[i] : nullptr, n);
    load_param(sw[i], a.post ? a.post + col[i] : nullptr, n);
    load_param(scale, a.scale ? a.scale + col[i] : nullptr, n);
#pragma unroll
    for (int e = 0; e < VL; ++e) sw[i][e] *= scale[e];
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
    for (int i = 0; i < NIT; ++i) {
#pragma unroll
      for (int e = 0; e < VL; ++e) {
        n1[i][e] = value(px[i], e);
        nw[i][e] = value(pr[i], e);
        if (BWD) {
          d[i][e] = value(pd[i], e);
          dn[i][e] = value(pn[i], e);
        }
        sum1[0] = fmaf(n1[i][e], n1[i][e], sum1[0]);
      }
    }
    fetch(row + step);
    float inv1 = 1.0f;
    if (a.post) {
      unit_sum<TPU>(sum1, turn);
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
    unit_sum<TPU>(sum2, turn);
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
        unit_sum<TPU>(sum3, turn);
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
    const int64_t slots = (int64_t)gridDim.x * U, slot = blockIdx.x * U + threadIdx.x / TPU;
    if (a.weight) write_columns<TPU>(dw, a.partial + slot * a.width, a.width);
    if (a.post || a.scale) write_columns<TPU>(db, a.partial + (slots + slot) * a.width, a.width);
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

template <int N>
using Int = std::integral_constant<int, N>;

// The unit that holds a row. Forward: one piece a thread (two beyond 1024 pieces, which only fp32 rows have), which keeps
// the registers few and a single row's latency short: against a wave with three pieces a thread, 1536 bf16 columns went
// from 13 to 4 us for 8 rows and from 208 to 178 us (4.5 TB/s) for 65536. Backward, with three sums one after the other in
// a row, barriers cost more than registers: waves of up to three pieces a thread, 254 us (4.7 TB/s) against 432 for 65536 rows of
// 1536 columns, then the fewest waves with two.
template <typename T, bool BWD, typename F>
void by_width(int64_t width, F f) {
  constexpr int VL = 16 / sizeof(T);
  const int64_t pieces = (width + VL - 1) / VL;
  if (pieces <= 16) return f(Int<16>{}, Int<1>{});
  if (pieces <= 32) return f(Int<32>{}, Int<1>{});
  if (pieces <= 64) return f(Int<64>{}, Int<1>{});
  if constexpr (BWD) {
    if (pieces <= 128) return f(Int<64>{}, Int<2>{});
    if (pieces <= 192) return f(Int<64>{}, Int<3>{});
    if (pieces <= 256) return f(Int<128>{}, Int<2>{});
    if (pieces <= 512) return f(Int<256>{}, Int<2>{});
    if (VL == 8 || pieces <= 1024) return f(Int<512>{}, Int<2>{});
  } else {
    if (pieces <= 128) return f(Int<128>{}, Int<1>{});
    if (pieces <= 192) return f(Int<192>{}, Int<1>{});
    if (pieces <= 256) return f(Int<256>{}, Int<1>{});
    if (pieces <= 384) return f(Int<384>{}, Int<1>{});
    if (pieces <= 512) return f(Int<512>{}, Int<1>{});
    if (pieces <= 768) return f(Int<768>{}, Int<1>{});
    if (VL == 8 || pieces <= 1024) return f(Int<1024>{}, Int<1>{});
  }
  if constexpr (VL == 4) f(Int<1024>{}, Int<2>{});
}

int64_t gcd(int64_t a, int64_t b) { return b == 0 ? a : gcd(b, a % b); }

// Workgroups of a launch over rows x groups units, U of them a workgroup: what every CU holds at once (backward, where each
// unit leaves a row of column sums: 1024, 512 or 256 threads by the pieces a thread has), and a multiple of the groups in
// units.
int64_t row_blocks(int64_t rows, int64_t groups, int tpu, int nit, bool backward) {
  const int64_t block = block_of(tpu), U = block / tpu, unit = groups / gcd(groups, U);  // blocks whose units are whole rows
  int64_t n = (int64_t)device_cus() * (!backward ? 2048 : nit == 1 ? 1024 : nit == 2 ? 512 : 256) / block;
  if (n < device_cus()) n = device_cus();
  const int64_t need = (rows * groups + U - 1) / U;
  if (n > need) n = need;
  return (n + unit - 1) / unit * unit;
}

int norm_status(int64_t rows, int64_t groups, int64_t width, int dtype) {
  if (rows < 0 || groups < 1 || width < 1) return TSF_ERR_ARG;
  if (dtype != TSF_DTYPE_F32 && dtype != TSF_DTYPE_BF16) return TSF_ERR_ARG;
  if (width > kMaxWidth || groups > 65535 || groups * width > INT32_MAX || rows > ((int64_t)1 << 31)) return TSF_ERR_UNSUPPORTED;
  return TSF_OK;
}

// Launches; the units there were (rows of the column sums, times the groups).
template <typename T, bool BWD>
int64_t gated(const GatedArgs& a, hipStream_t stream) {
  int64_t units = 0;
  by_width<T, BWD>(a.width, [&](auto tpu, auto nit) {
    constexpr int TPU = decltype(tpu)::value, NIT = decltype(nit)::value;
    const int64_t blocks = row_blocks(a.rows, a.groups, TPU, NIT, BWD);
    gated_kernel<T, TPU, NIT, BWD><<<(unsigned)blocks, block_of(TPU), 0, stream>>>(a);
    units = blocks * (block_of(TPU) / TPU);
  });
  return units;
}

template <typename T, typename R, bool BWD>
int64_t residual(const ResidualArgs& a, hipStream_t stream) {
  int64_t units = 0;
  by_width<T, BWD>(a.width, [&](auto tpu, auto nit) {
    constexpr int TPU = decltype(tpu)::value, NIT = decltype(nit)::value;
    const int64_t blocks = row_blocks(a.rows, 1, TPU, NIT, BWD);
    residual_kernel<T, R, TPU, NIT, BWD><<<(unsigned)blocks, block_of(TPU), 0, stream>>>(a);
    units = blocks * (block_of(TPU) / TPU);
  });
  return units;
}

// Bytes of the column sums of `sums` parameters, whichever type the rows have.
int64_t partial_bytes(int64_t rows, int64_t groups, int64_t width, int sums) {
  int64_t most = 0;
  auto take = [&](auto tpu, auto nit) {
    constexpr int TPU = decltype(tpu)::value, NIT = decltype(nit)::value;
    const int64_t n = row_blocks(rows, groups, TPU, NIT, true) * (block_of(TPU) / TPU);
    if (n > most) most = n;
  };
  by_width<float, true>(width, take);
  by_width<bf16, true>(width, take);
  return most * width * sums * 4;
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
  return partial_bytes(rows, groups, width, 1);
}

int64_t tsfast_hip_residual_norm_workspace_bytes(int64_t rows, int64_t width) {
  if (norm_status(rows, 1, width, TSF_DTYPE_F32) != TSF_OK) return -1;
  return partial_bytes(rows, 1, width, 2);
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
  const int64_t units = dtype == TSF_DTYPE_BF16 ? gated<bf16, true>(a, st) : gated<float, true>(a, st);
  if (weight) reduce(a.partial, (int)(units / groups), groups * width, grad_weight, nullptr, nullptr, nullptr, st);
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
  const int blocks = (int)(dtype == TSF_DTYPE_F32        ? residual<float, float, true>(a, st)
                           : res_dtype == TSF_DTYPE_BF16 ? residual<bf16, bf16, true>(a, st)
                                                         : residual<bf16, float, true>(a, st));
  if (weight) reduce(a.partial, blocks, width, grad_weight, nullptr, nullptr, nullptr, st);
  if (post_weight || scale)
    reduce(a.partial + (int64_t)blocks * width, blocks, width, post_weight ? grad_post_weight : nullptr, scale, scale ? grad_scale : nullptr, post_weight,
           st);
  return tsf_launch_status();
}

}  // extern "C"
