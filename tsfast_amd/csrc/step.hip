// A Mamba layer for one token of each sequence: all that stands between its input and its output projection (gfx950).
//
//   u = silu(bias + conv weight . (tail, x))                 tail <- its last K - 1 inputs
//   (dt, B, C) = x_proj u,  delta = softplus(dt_proj dt + dt_bias)
//   h <- exp(delta A) h + delta u B,  out = (h C + Dp u) silu(z)
//
// Two launches. project_kernel forms u, moves the convolution's state and multiplies u by x_proj, slice by slice of the channels;
// advance_kernel adds the slices' sums, forms delta and moves the scan's state, in place. Everything in between is float32. Products
// with float32 parameters are float32 matrix instructions; with bfloat16 ones the float32 factor goes in as three bfloat16 parts, exact to
// 2^-24, on the bfloat16 matrix cores (48 cycles for 32 channels instead of 256).
#include <type_traits>

#include "common.h"
#include "tsfast_hip.h"

using namespace tsf;

namespace {

constexpr int kThreads = 256;
constexpr int kCh = 64;     // channels of a step of a slice, and of a workgroup of advance_kernel
constexpr int kRowsP = 16;  // rows (sequences) of a workgroup of project_kernel
constexpr int kRowsA = 8;   // and of advance_kernel
constexpr int kMaxK = 8, kMaxN = 64;
constexpr int64_t kMaxP = 1024;  // R + 2 N

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct StepArgs {
  const void *x, *z;
  void *tail, *out;
  float* h;
  const void *wc, *bc, *xp, *dp, *db;  // conv weight and bias, x_proj, dt_proj, dt_bias
  const float *A, *Dp;
  int64_t B, D, sx, sz, slice;  // slice: channels
  int N, R, P, K, slices, db16;
  float *part, *u;  // [slices][B][P]; [B][D]
};

// Loads are unconditional, from clamped addresses, and what does not exist is made zero behind them: a load under a condition of its own
// is waited for before the next one starts, and these kernels are chains of latencies.

// 8 values of a row at any alignment as they lie, and as floats: the first n of them, zeros after. whole: there are 8 behind p wherever n > 0
// (and behind p where n <= 0, whatever they are)
template <typename P>
struct Eight {
  P h[8];
  TSF_DEV void load(const P* p, int n, bool whole) {
    if (whole) {
      __builtin_memcpy(h, p, sizeof(h));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] = e < n ? p[e] : from_f32<P>(0.0f);
    }
  }
  // what there is not of 8, made zero
  TSF_DEV void fit(int n) {
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = e < n ? h[e] : from_f32<P>(0.0f);
  }
};

// The other factor of a product: ROWS rows of floats in LDS, `cols` a row, 8 of them a lane at once.
template <typename P, int ROWS>
struct Side;
template <int ROWS>
struct Side<float, ROWS> {
  char* at;
  int stride;  // elements
  static constexpr int bytes(int cols) { return ROWS * (cols + 4) * 4; }
  TSF_DEV Side(char* lds, int cols) : at(lds), stride(cols + 4) {}
  TSF_DEV void put(int row, int col, float v) const { ((float*)at)[row * stride + col] = v; }
  template <int N>
  TSF_DEV void multiply(const Eight<float>* w, int row, int col, f32x4* acc) const {
    float v[8];
    __builtin_memcpy(v, __builtin_assume_aligned(at + (row * stride + col) * 4, 16), 32);
#pragma unroll
    for (int e = 0; e < 8; ++e)
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(w[i].h[e], v[e], acc[i], 0, 0, 0);
  }
};
template <int ROWS>
struct Side<bf16, ROWS> {
  char* at;
  int stride;
  static constexpr int bytes(int cols) { return 3 * ROWS * (cols + 8) * 2; }
  TSF_DEV Side(char* lds, int cols) : at(lds), stride(cols + 8) {}
  TSF_DEV void put(int row, int col, float v) const {
    bf16* p = (bf16*)at + row * stride + col;
    // at most bf16's largest at first: a float above it is the sum of its parts too, an infinity (bf16's largest, itself, itself)
    constexpr float kMost = 3.3895314e38f;
    const bf16 first = from_f32<bf16>(fminf(fmaxf(v, -kMost), kMost));
    const float rest = v - to_f32(first);
    const bf16 second = from_f32<bf16>(rest);
    const float last = rest - to_f32(second);
    p[0] = first;
    p[ROWS * stride] = second;
    p[2 * ROWS * stride] = from_f32<bf16>(last == last ? last : rest);
  }
  template <int N>
  TSF_DEV void multiply(const Eight<bf16>* w, int row, int col, f32x4* acc) const {
#pragma unroll
    for (int n = 2; n >= 0; --n) {  // the least part first
      bf16x8 v;
      __builtin_memcpy(&v, __builtin_assume_aligned((bf16*)at + (n * ROWS + row) * stride + col, 16), 16);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        bf16x8 f;
        __builtin_memcpy(&f, w[i].h, 16);
        acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, v, acc[i], 0, 0, 0);
      }
    }
  }
};

// What u of one channel of one row is made of. K taps; K = 0: any number up to 8, by g.K.
template <typename T, typename P, int K>
struct Window {
  static constexpr int kTaps = K ? K : kMaxK;
  T past[kTaps];  // the last one is x
  P w[kTaps], bias;
  TSF_DEV static int taps(const StepArgs& g) { return K ? K : g.K; }
  TSF_DEV void load(const StepArgs& g, int64_t b, int64_t d) {
    const int n = taps(g);
    const T* tail = (const T*)g.tail + (b * g.D + d) * (n - 1);
    const P *wc = (const P*)g.wc + d * n, *bc = g.bc ? (const P*)g.bc + d : wc;
    bias = *bc;
    past[kTaps - 1] = ((const T*)g.x)[b * g.sx + d];
#pragma unroll
    for (int k = 0; k < kTaps; ++k) {
      const int i = k < n ? k : n - 1;
      w[k] = wc[i];
      if (k + 1 < kTaps) past[k] = tail[k < n - 1 ? k : n - 2];
    }
  }
  TSF_DEV float u(const StepArgs& g) const {
    const int n = taps(g);
    float a = g.bc ? to_f32(bias) : 0.0f;
#pragma unroll
    for (int k = 0; k + 1 < kTaps; ++k) a = k < n - 1 ? fmaf(to_f32(w[k]), to_f32(past[k]), a) : a;
    a = fmaf(to_f32(w[kTaps - 1]), to_f32(past[kTaps - 1]), a);  // w[kTaps - 1] is the last tap's, whatever n is
    return a * sigmoid_fast(a);
  }
  TSF_DEV void move(const StepArgs& g, int64_t b, int64_t d) const {
    const int n = taps(g);
    T* tail = (T*)g.tail + (b * g.D + d) * (n - 1);
#pragma unroll
    for (int k = 0; k + 1 < kTaps; ++k)
      if (k < n - 1) tail[k] = k + 1 < n - 1 ? past[k + 1 < kTaps - 1 ? k + 1 : k] : past[kTaps - 1];
  }
};

// A workgroup: 16 rows, one slice of the channels, x_proj's columns 128 at a time, 32 a wave. Lane group lg has channels 8 lg .. of each 32.
// u goes out and the convolution's state moves on with the last columns.
template <typename T, typename P, int K>
__global__ void __launch_bounds__(kThreads) project_kernel(StepArgs g) {
  __shared__ __attribute__((aligned(16))) char s_u[Side<P, kRowsP>::bytes(kCh)];
  const Side<P, kRowsP> side(s_u, kCh);
  const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, lg = lane >> 4, wave = tid >> 6;
  const int64_t slice = blockIdx.x % g.slices, b0 = blockIdx.x / g.slices * kRowsP;
  const int64_t c_begin = slice * g.slice, c_end = c_begin + g.slice < g.D ? c_begin + g.slice : g.D;
  constexpr int kTiles = 2;              // of 16 columns that a wave has at once
  constexpr int kOwn = kRowsP / 4;       // rows of its channel that a thread owns: wave + 4 i
  constexpr int kColumns = 4 * 16 * kTiles;
  for (int p0 = 0; p0 < g.P; p0 += kColumns) {
    const bool last = p0 + kColumns >= g.P;
    f32x4 acc[kTiles];
#pragma unroll
    for (int i = 0; i < kTiles; ++i) acc[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // a step's inputs are loaded while the one before is multiplied
    struct Inputs {
      Window<T, P, K> win[kOwn];
      Eight<P> w[kCh / 32][kTiles];
    } next;
    auto load = [&](int64_t c) __attribute__((always_inline)) {
      const int64_t d = c + lane;
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        const int64_t b = b0 + wave + 4 * i;
        next.win[i].load(g, b < g.B ? b : g.B - 1, d < c_end ? d : c_end - 1);
      }
      const bool whole = c + kCh <= c_end;
#pragma unroll
      for (int k = 0; k < kCh / 32; ++k)
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
          const int64_t at = c + 32 * k + 8 * lg;
          const int p = p0 + (wave * kTiles + i) * 16 + li;
          next.w[k][i].load((const P*)g.xp + (int64_t)(p < g.P ? p : g.P - 1) * g.D + at, c_end > at ? (int)(c_end - at < 8 ? c_end - at : 8) : 0, whole);
        }
    };
    load(c_begin);
    for (int64_t c = c_begin; c < c_end; c += kCh) {
      const int64_t d = c + lane;
      const Inputs now = next;
      if (c > c_begin || p0 > 0) __syncthreads();  // the step before has been read
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        const int r = wave + 4 * i;
        const bool in = b0 + r < g.B && d < c_end;
        const float u = now.win[i].u(g);
        side.put(r, lane, in ? u : 0.0f);
        if (in && last) {
          now.win[i].move(g, b0 + r, d);
          g.u[(b0 + r) * g.D + d] = u;
        }
      }
      if (c + kCh < c_end) load(c + kCh);
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kCh / 32; ++k) side.template multiply<kTiles>(now.w[k], li, 32 * k + 8 * lg, acc);
    }
    // columns 4 lg + e of row li
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      const int p = p0 + (wave * kTiles + i) * 16 + 4 * lg;
      if (b0 + li < g.B) {
        float* to = g.part + (slice * g.B + b0 + li) * g.P + p;
        if (g.P % 4 == 0) {
          if (p < g.P) __builtin_memcpy(to, &acc[i], 16);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (p + e < g.P) to[e] = acc[i][e];
        }
      }
    }
  }
}

// A workgroup: 64 channels of up to 8 rows. States: 4 lanes a channel, 4 states of each 16 a lane. delta: 16 channels a wave.
// Three waves a SIMD, for three workgroups a CU: 256 sequences of 1536 channels 15.7 us, with two (180 registers) 4 more, with four (which
// spill) 8.
template <typename T, typename P, int NV>
__global__ void __launch_bounds__(kThreads, NV == 1 ? 3 : 2) advance_kernel(StepArgs g) {
  extern __shared__ __attribute__((aligned(16))) char s_dt[];  // [rows][R], zeros up to a multiple of 32
  __shared__ __attribute__((aligned(16))) float s_bc[2][kRowsA][16 * NV];  // B and C
  __shared__ float4 s_c[kRowsA][kCh + 1];  // delta, delta u, Dp u, silu(z)
  const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, lg = lane >> 4, wave = tid >> 6;
  const int64_t tiles = (g.D + kCh - 1) / kCh, tile = blockIdx.x % tiles, b0 = blockIdx.x / tiles * kRowsA;
  const int rows = (int)(g.B - b0 < kRowsA ? g.B - b0 : kRowsA);
  const int N = g.N, R = g.R, R32 = (R + 31) / 32 * 32, columns = g.P;
  const Side<P, kRowsA> side(s_dt, R32);

  // Loads return in order: the slices' sums first, for all that follows waits for them; the states stream in behind.
  constexpr int kSums = 4, kSlices = 8;  // columns of rows that a thread sums at once, slices that it loads at once
  const int count = rows * columns;
  const int64_t stride = g.B * columns;
  const float* part = g.part + b0 * columns;
  float v[kSums][kSlices];
  auto load_sums = [&](int i0, int k0) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < kSlices; ++k)
#pragma unroll
      for (int q = 0; q < kSums; ++q) {
        const int i = i0 + q * kThreads;
        v[q][k] = part[(k0 + k < g.slices ? k0 + k : 0) * stride + (i < count ? i : 0)];
      }
  };
  load_sums(tid, 0);
  // the first of dt_proj's values, whose channel this lane brings
  const int64_t dw = tile * kCh + 16 * wave + li;
  const P* wrow = (const P*)g.dp + (dw < g.D ? dw : g.D - 1) * R;
  const bool whole = R % 8 == 0;
  constexpr int kFirst = sizeof(P) == 2 ? 4 : 2;
  Eight<P> w[kFirst];
#pragma unroll
  for (int k = 0; k < kFirst; ++k) w[k].load(wrow + (32 * k + 8 * lg < R ? 32 * k + 8 * lg : 0), R - 32 * k - 8 * lg, whole);
  // this lane's part of delta: channels d .. d + 3 of row li
  const int64_t d = tile * kCh + 16 * wave + 4 * lg, b = b0 + (li < rows ? li : rows - 1);
  const bool row = li < rows;
  float u[4], dp[4], bias[4];
  T z[4];
  if (g.D % 4 == 0) {
    const int64_t i = d < g.D ? d : g.D - 4;
    __builtin_memcpy(u, g.u + b * g.D + i, 16);
    __builtin_memcpy(z, (const T*)g.z + b * g.sz + i, sizeof(z));
    __builtin_memcpy(dp, g.Dp + i, 16);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int64_t i = d + e < g.D ? d + e : g.D - 1;
      u[e] = g.u[b * g.D + i], z[e] = ((const T*)g.z)[b * g.sz + i], dp[e] = g.Dp[i];
    }
  }
  if (!g.db) {
#pragma unroll
    for (int e = 0; e < 4; ++e) bias[e] = 0.0f;
  } else if (g.db16) {
#pragma unroll
    for (int e = 0; e < 4; ++e) bias[e] = to_f32(((const bf16*)g.db)[d + e < g.D ? d + e : g.D - 1]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) bias[e] = ((const float*)g.db)[d + e < g.D ? d + e : g.D - 1];
  }
  // the states
  const int q = tid & 3;
  const int64_t dh = tile * kCh + (tid >> 2);
  const bool act = dh < g.D;
  const bool full = N == 16 * NV;  // every lane's states exist
  constexpr int kAhead = NV == 1 ? kRowsA : 2;  // rows whose states are read ahead
  f32x4 h[kAhead][NV];
  auto load4 = [&](f32x4* to, const float* p) __attribute__((always_inline)) {
    if (full) {
#pragma unroll
      for (int j = 0; j < NV; ++j) __builtin_memcpy(&to[j], p + 16 * j + 4 * q, 16);
    } else {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) to[j][e] = 16 * j + 4 * q + e < N ? p[16 * j + 4 * q + e] : 0.0f;
    }
  };
  auto load_state = [&](f32x4* to, int r) __attribute__((always_inline)) {
    load4(to, g.h + ((b0 + (r < rows ? r : rows - 1)) * g.D + (act ? dh : g.D - 1)) * N);
  };
  f32x4 A2[NV];
  load4(A2, g.A + (act ? dh : g.D - 1) * N);
#pragma unroll
  for (int r = 0; r < kAhead; ++r) load_state(h[r], r);

  for (int i = tid; i < kRowsA * (R32 - R); i += kThreads) side.put(i / (R32 - R), R + i % (R32 - R), 0.0f);
  for (int i = tid; i < 2 * kRowsA * (16 * NV - N); i += kThreads) (&s_bc[0][0][0])[i / (16 * NV - N) * (16 * NV) + N + i % (16 * NV - N)] = 0.0f;
  for (int i0 = tid;;) {
    float s[kSums] = {};
    for (int k0 = 0;;) {
#pragma unroll
      for (int k = 0; k < kSlices; ++k)
#pragma unroll
        for (int n = 0; n < kSums; ++n) s[n] += k0 + k < g.slices ? v[n][k] : 0.0f;
      k0 += kSlices;
      if (k0 >= g.slices) break;
      load_sums(i0, k0);
    }
#pragma unroll
    for (int n = 0; n < kSums; ++n) {
      const int i = i0 + n * kThreads, r = i / columns, c = i % columns;
      if (i < count) {
        if (c < R)
          side.put(r, c, s[n]);
        else
          s_bc[c >= R + N][r][c < R + N ? c - R : c - R - N] = s[n];
      }
    }
    i0 += kSums * kThreads;
    if (i0 - tid >= count) break;
    load_sums(i0, 0);
  }
  __syncthreads();
  {
    f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    const int from = li < kRowsA ? li : li - kRowsA;  // rows that do not exist: any, their columns are not used
#pragma unroll
    for (int k = 0; k < kFirst; ++k)
      if (32 * k < R) {
        w[k].fit(R - 32 * k - 8 * lg);
        side.template multiply<1>(&w[k], from, 32 * k + 8 * lg, &acc);
      }
    for (int k = 32 * kFirst; k < R; k += 32) {
      Eight<P> f;
      f.load(wrow + (k + 8 * lg < R ? k + 8 * lg : 0), R - k - 8 * lg, whole);
      f.fit(R - k - 8 * lg);
      side.template multiply<1>(&f, from, k + 8 * lg, &acc);
    }
    if (row) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float delta = softplus_fast(acc[e] + bias[e]), zz = to_f32(z[e]);
        s_c[li][16 * wave + 4 * lg + e] = make_float4(delta, delta * u[e], dp[e] * u[e], zz * sigmoid_fast(zz));
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) A2[j] *= kLog2e;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRowsA; ++r) {
    if (r < rows) {
      f32x4* hr = h[r % kAhead];
      const float4 c = s_c[r][tid >> 2];
      float y = 0.0f;
      float* p = g.h + ((b0 + r) * g.D + dh) * N + 4 * q;
      auto advance = [&](auto all) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          const f32x4 Bt = *(const f32x4*)&s_bc[0][r][16 * j + 4 * q], Ct = *(const f32x4*)&s_bc[1][r][16 * j + 4 * q];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            // states that do not exist stay out: zeros, but for an infinite delta, with which their products are NaN
            const float to = fmaf(fast_exp2(c.x * A2[j][e]), hr[j][e], c.y * Bt[e]);
            hr[j][e] = all || 16 * j + 4 * q + e < N ? to : 0.0f;
            y = fmaf(hr[j][e], Ct[e], y);
          }
          if (act) {
            if (all) {
              __builtin_memcpy(p + 16 * j, &hr[j], 16);
            } else {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (16 * j + 4 * q + e < N) p[16 * j + e] = hr[j][e];
            }
          }
        }
      };
      if (full)
        advance(std::true_type());
      else
        advance(std::false_type());
      if (kAhead < kRowsA && r + kAhead < kRowsA) load_state(hr, r + kAhead);
      y += __shfl_xor(y, 1, kWave);
      y += __shfl_xor(y, 2, kWave);
      if (q == 0 && act) ((T*)g.out)[(b0 + r) * g.D + dh] = from_f32<T>((y + c.z) * c.w);
    }
  }
}

// ------------------------------------------------------------------------------------------ host
int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }
constexpr int64_t kMaxGrid = (1 << 24) - 1;

// Channels of a slice: enough slices for half a workgroup a CU. More of them would be read again by each of advance_kernel's workgroups.
int64_t slice_for(int64_t B, int64_t D) {
  const int64_t steps = up(D, kCh), slices = up((int64_t)device_cus() / 2, up(B, kRowsP));
  return (slices >= steps ? 1 : up(steps, slices)) * kCh;
}

int step_status(int64_t B, int64_t D, int64_t N, int64_t R, int64_t K) {
  if (B < 0 || D < 0 || N < 1 || R < 1 || K < 2) return TSF_ERR_ARG;
  if (K > kMaxK || N > kMaxN || R + 2 * N > kMaxP || D > (int64_t)1 << 24 || B > (int64_t)1 << 31) return TSF_ERR_UNSUPPORTED;
  if (up(B, kRowsA) * up(D, kCh) > kMaxGrid) return TSF_ERR_UNSUPPORTED;
  return TSF_OK;
}

template <typename T, typename P, int K>
void launch_project(const StepArgs& a, hipStream_t st) {
  project_kernel<T, P, K><<<(unsigned)(up(a.B, kRowsP) * a.slices), kThreads, 0, st>>>(a);
}
template <typename T, typename P>
void launch_step(const StepArgs& a, hipStream_t st) {
  switch (a.K) {
    case 2: launch_project<T, P, 2>(a, st); break;
    case 3: launch_project<T, P, 3>(a, st); break;
    case 4: launch_project<T, P, 4>(a, st); break;
    default: launch_project<T, P, 0>(a, st); break;
  }
  const unsigned grid = (unsigned)(up(a.B, kRowsA) * up(a.D, kCh));
  const size_t lds = (size_t)Side<P, kRowsA>::bytes((int)up(a.R, 32) * 32);
  if (a.N <= 16)
    advance_kernel<T, P, 1><<<grid, kThreads, lds, st>>>(a);
  else if (a.N <= 32)
    advance_kernel<T, P, 2><<<grid, kThreads, lds, st>>>(a);
  else
    advance_kernel<T, P, 4><<<grid, kThreads, lds, st>>>(a);
}

}  // namespace

extern "C" {

int64_t tsfast_hip_mamba_step_workspace_bytes(int64_t B, int64_t D, int64_t N, int64_t R, int64_t K) {
  if (step_status(B, D, N, R, K) != TSF_OK) return -1;
  if (B == 0 || D == 0) return 0;
  return (up(D, slice_for(B, D)) * (R + 2 * N) + D) * B * 4;
}

int tsfast_hip_mamba_step(int64_t B, int64_t D, int64_t N, int64_t R, int64_t K, int io_dtype, int param_dtype, int dt_bias_dtype, const void* x,
                          int64_t x_stride, const void* z, int64_t z_stride, void* conv_state, float* ssm_state, const void* conv_weight,
                          const void* conv_bias, const void* x_proj, const void* dt_proj, const void* dt_bias, const float* A,
                          const float* Dp, void* out, void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = step_status(B, D, N, R, K);
  if (rc != TSF_OK) return rc;
  for (const int t : {io_dtype, param_dtype, dt_bias_dtype})
    if (t != TSF_DTYPE_F32 && t != TSF_DTYPE_BF16) return TSF_ERR_ARG;
  if (x_stride < 0 || z_stride < 0) return TSF_ERR_ARG;
  if (B == 0 || D == 0) return TSF_OK;
  if (!x || !z || !conv_state || !ssm_state || !conv_weight || !x_proj || !dt_proj || !A || !Dp || !out) return TSF_ERR_ARG;
  if (!workspace || workspace_bytes < tsfast_hip_mamba_step_workspace_bytes(B, D, N, R, K)) return TSF_ERR_WORKSPACE;
  StepArgs a = {};
  a.x = x, a.z = z, a.tail = conv_state, a.out = out, a.h = ssm_state, a.wc = conv_weight, a.bc = conv_bias, a.xp = x_proj, a.dp = dt_proj;
  a.db = dt_bias, a.A = A, a.Dp = Dp, a.B = B, a.D = D, a.sx = x_stride, a.sz = z_stride, a.slice = slice_for(B, D);
  a.N = (int)N, a.R = (int)R, a.P = (int)(R + 2 * N), a.slices = (int)up(D, a.slice), a.part = (float*)workspace;
  a.K = (int)K, a.db16 = dt_bias_dtype == TSF_DTYPE_BF16, a.u = a.part + a.slices * B * a.P;
  const hipStream_t st = (hipStream_t)stream;
  if (io_dtype == TSF_DTYPE_BF16 && param_dtype == TSF_DTYPE_BF16)
    launch_step<bf16, bf16>(a, st);
  else if (io_dtype == TSF_DTYPE_BF16)
    launch_step<bf16, float>(a, st);
  else if (param_dtype == TSF_DTYPE_BF16)
    launch_step<float, bf16>(a, st);
  else
    launch_step<float, float>(a, st);
  return tsf_launch_status();
}

}  // extern "C"
