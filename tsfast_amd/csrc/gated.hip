// Gated linear recurrence with a matrix state per head (gfx950).
//
//   S_t = exp(g_t) S_{t-1} + k_t v_t^T,   o_t = S_t^T q_t
//
// and, with T_t = dL/dS_t running backwards (T_t = exp(g_{t+1}) T_{t+1} + q_t do_t^T),
//
//   dq_t = S_t do_t,   dk_t = T_t v_t,   dv_t = T_t^T k_t,   dg_t = exp(g_t) <S_{t-1}, T_t>.
//
// The output and the three gradients are one form. With G the running sum of g and
// D(a, b) = exp(G_a - G_b),
//
//   out_i = sum_j D x_i . y_j z_j     forward in time (j <= i):   o (q, k, v),  dq (do, v, k)
//                                     backward in time (j >= i):  dv (k, q, do), dk (v, do, q)
//
// so one kernel, walk_kernel, computes all four. A workgroup owns one head of one row, a tile of FT of z's
// columns and a run of 64-step chunks; the state tile stays in fp32 accumulator registers from the first
// chunk to the last and is never written in between. Per chunk the decayed scores of x and y within
// it (64 x 64, the causal half only) times z, x times the state before it, and the state's update are MFMA
// products; the decays come from exact differences of a float64 running sum, so any g <= 0 down to -inf
// keeps its accuracy.
//
// dg needs no product of its own: r_t = q_t . dq_t and c_t = k_t . dk_t, summed while dq and dk are still in
// registers, give dg_{t+1} = dg_t - r_t + c_t. The rounding errors of that running sum are cut off at
// anchors every kAnchor chunks, where dg_t = <S_{t-1}, dL/dS_{t-1}> is formed from the two states.
#include <type_traits>

#include "common.h"
#include "tsfast_hip.h"

using namespace tsf;

namespace {

constexpr int kC = 64;          // steps of a chunk
constexpr int kThreads = 256;   // four waves; wave w owns the chunk's steps 16 w .. 16 w + 15
constexpr int kFT = 64;         // columns of z a workgroup owns
constexpr int kMaxWidth = 128;  // of K and V
constexpr int kStepMaxK = 1024;  // of K in a single step
constexpr int kMaxGrid = (1 << 24) - 1;
// log2 decay that stands for all smaller ones, -inf among them: 2^-300 is zero in fp32, and sums of
// 64 such gates keep 1e-11 in their float64 sums
constexpr double kNoDecayLeft = -300.0;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// An operand of a 16 x 16 product: 8 values of one row along the contraction, which lane group
// lane >> 4 holds; the row is lane & 15. Both operands have the same layout, so any order of the
// contraction will do as long as both have it.
template <typename T>
struct Frag;
template <>
struct Frag<bf16> {
  bf16x8 v;
};
template <>
struct Frag<float> {
  f32x4 lo, hi;
};

TSF_DEV f32x4 mma(const Frag<bf16>& a, const Frag<bf16>& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0);
}
TSF_DEV f32x4 mma(const Frag<float>& a, const Frag<float>& b, f32x4 c) {
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.lo[e], b.lo[e], c, 0, 0, 0);
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.hi[e], b.hi[e], c, 0, 0, 0);
  return c;
}

TSF_DEV float get(const Frag<bf16>& f, int e) { return (float)f.v[e]; }
TSF_DEV float get(const Frag<float>& f, int e) { return e < 4 ? f.lo[e & 3] : f.hi[e & 3]; }
TSF_DEV void put(Frag<bf16>& f, int e, float x) { f.v[e] = (__bf16)x; }
TSF_DEV void put(Frag<float>& f, int e, float x) {
  if (e < 4)
    f.lo[e & 3] = x;
  else
    f.hi[e & 3] = x;
}

// Eight values as the sum of N operands: bf16 carries 8 bits of each value's mantissa an operand, fp32 all.
template <typename T, int N>
TSF_DEV void split(const float* x, Frag<T>* out) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float rest = x[e];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      put(out[n], e, rest);
      if (n + 1 < N) rest -= get(out[n], e);
    }
  }
}

// Eight consecutive values of a row of global memory at any alignment; `n` of them exist.
TSF_DEV void load8(Frag<bf16>& f, const bf16* p, int n) {
  if (n >= 8) {
    __builtin_memcpy(&f.v, p, 16);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      f.v[e] = (__bf16)0.0f;
      if (e < n) f.v[e] = __builtin_bit_cast(__bf16, p[e].bits);
    }
  }
}
TSF_DEV void load8(Frag<float>& f, const float* p, int n) {
  if (n >= 8) {
    __builtin_memcpy(&f.lo, p, 16);
    __builtin_memcpy(&f.hi, p + 4, 16);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) put(f, e, e < n ? p[e] : 0.0f);
  }
}
// Four consecutive values of a row of global memory at any alignment; `n` of them exist.
TSF_DEV void store4(float* p, f32x4 v, int n) {
  if (n >= 4) {
    __builtin_memcpy(p, &v, 16);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) p[e] = v[e];
  }
}
TSF_DEV void store4(bf16* p, f32x4 v, int n) {
  bf16 h[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) h[e] = from_f32<bf16>(v[e]);
  if (n >= 4) {
    __builtin_memcpy(p, h, 8);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) p[e] = h[e];
  }
}
TSF_DEV f32x4 load4(const float* p, int n) {
  f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  if (n >= 4) {
    __builtin_memcpy(&v, p, 16);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) v[e] = p[e];
  }
  return v;
}
TSF_DEV f32x4 load4(const bf16* p, int n) {
  f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  bf16 h[4];
  if (n >= 4) {
    __builtin_memcpy(h, p, 8);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = to_f32(h[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) v[e] = to_f32(p[e]);
  }
  return v;
}

// A sequence tensor: strides in elements of the batch row, the step and the head; `share` heads of the
// state read one head of it. The innermost dimension is dense.
template <typename T>
struct Seq {
  T* p;
  int64_t sb, sl, sh;
  int share;
  TSF_DEV T* row(int64_t b, int64_t t, int h) const { return p + b * sb + t * sl + (int64_t)(h / share) * sh; }
};

template <typename T, typename OT>
struct WalkArgs {
  Seq<const T> x, y, z, g;
  Seq<OT> out;
  int H, E, F;       // heads, columns of x and y, columns of z
  int64_t L, units;  // steps; rows x heads x segments
  int nft, nseg, seg_chunks;
  int se, sf;                // strides of a state's element (e, f)
  const float* init;         // state entering each unit [row x head (x segment)][K V]; null: zero
  int init_per_seg;          // whether init holds one for each segment
  float* last;               // state leaving: of the row, [row x head][K V], or of the segment (state_only)
  double* seg_decay;         // state_only: log2 of the segment's decay
  Seq<const T> dot;          // out_i . dot_i is summed over this tile's columns ..
  float* dots;               // .. into [tile][row x head][L]
  float* anchors;            // states before every anchor chunk [row x head][anchor][K V]: written forward, read backward
  float* anchor_dots;        // backward: <state, anchor> over this tile [tile][row x head][anchor]
  int anchor_chunks, nanchor;
};

template <typename T, int E>
struct Lds {
  static constexpr bool kBf = sizeof(T) == 2;
  static constexpr int kRow = E + (kBf ? 8 : 4);  // pitch of Y and S rows: 16 bytes of padding against bank conflicts
  static constexpr int kCol = kC + 8;             // pitch of the transposed rows (bf16)
  static constexpr int kZRow = kFT + 4;           // pitch of z's rows (fp32)
  static constexpr int kSplit = kBf ? 2 : 1;      // operands the state is split into
  T y[kC * kRow];
  T yt[kBf ? E * kCol : 1];
  T z[kBf ? kFT * kCol : kC * kZRow];
  T s[kSplit][kFT * kRow];
  float hi[2][kC], lo[2][kC], w[2][kC], in[2][kC];  // running log2 decay, weights into the state and out of it
};

// Where step j of a chunk stands in a transposed row: an operand's 8 values (lane group lg, 32-step half s)
// are steps 32 s + 16 h + 4 lg + q in the order (h, q), the order the score tiles leave them in registers.
TSF_HOST_DEV int place(int j) { return (j & 32) + ((j >> 2) & 3) * 8 + ((j >> 4) & 1) * 4 + (j & 3); }

// One wave: the chunk's running log2 decay as float pairs (differences are exact to float64 rounding), the
// weight of each step in the state leaving the chunk, and of the state entering it at each step.
template <typename T, int E, bool FWD, typename A>
TSF_DEV void gates(Lds<T, E>& s, int buf, const A& a, int64_t b, int h, int64_t t0, int lane) {
  double G = 0.0;
  const int64_t t = t0 + lane;
  if (t < a.L) {
    const double x = (double)to_f32(*a.g.row(b, t, h)) * 1.4426950408889634;
    G = x < kNoDecayLeft ? kNoDecayLeft : x;  // NaN stays
  }
#pragma unroll
  for (int d = 1; d < kC; d <<= 1) {
    const double up = __shfl_up(G, d, kWave);
    if (lane >= d) G += up;
  }
  const double end = __shfl(G, kC - 1, kWave);
  const float hi = (float)G;
  s.hi[buf][lane] = hi;
  s.lo[buf][lane] = (float)(G - (double)hi);
  const float from = fast_exp2((float)G), to = fast_exp2((float)(end - G));
  s.in[buf][lane] = FWD ? from : to;
  s.w[buf][lane] = FWD ? to : from;
}

// Operand (row, k): 8 values at k of a row-major LDS array.
template <typename T>
TSF_DEV Frag<T> lds_row(const T* p) {
  Frag<T> f;
  __builtin_memcpy(&f, __builtin_assume_aligned(p, 16), sizeof(f));
  return f;
}
// Operand whose row is a column of y or z and whose contraction runs over steps (half s, lane group lg).
TSF_DEV Frag<bf16> lds_col(const bf16* t, int pitch, int col, int s, int lg) { return lds_row(t + col * pitch + 32 * s + 8 * lg); }
TSF_DEV Frag<float> lds_col(const float* t, int pitch, int col, int s, int lg) {
  Frag<float> f;
#pragma unroll
  for (int e = 0; e < 8; ++e) put(f, e, t[(32 * s + 16 * (e >> 2) + 4 * lg + (e & 3)) * pitch + col]);
  return f;
}

// A 4-step by 8-column piece of y or z on its way from global memory to LDS.
template <typename T>
struct Piece {
  Frag<T> r[4];
};
template <typename T>
TSF_DEV void fetch(Piece<T>& p, const Seq<const T>& q, int64_t b, int64_t t, int64_t L, int h, int col, int width) {
#pragma unroll
  for (int r = 0; r < 4; ++r) load8(p.r[r], q.row(b, t + r < L ? t + r : 0, h) + col, t + r < L ? width - col : 0);
}
template <typename T>
TSF_DEV void lds_rows(T* dst, int pitch, int j, int col, const Piece<T>& p) {
#pragma unroll
  for (int r = 0; r < 4; ++r)
    __builtin_memcpy(__builtin_assume_aligned(dst + (j + r) * pitch + col, 16), &p.r[r], sizeof(Frag<T>));
}
TSF_DEV void lds_cols(bf16* dst, int pitch, int j, int col, const Piece<bf16>& p) {
  const int at = place(j);
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    __bf16 v[4] = {p.r[0].v[c], p.r[1].v[c], p.r[2].v[c], p.r[3].v[c]};
    __builtin_memcpy(__builtin_assume_aligned(dst + (col + c) * pitch + at, 8), v, 8);
  }
}
TSF_DEV void lds_cols(float*, int, int, int, const Piece<float>&) {}

TSF_DEV float wave_sum(float x) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) x += __shfl_xor(x, m, kWave);
  return x;
}

// E: columns of x and y, padded; FWD: the direction in time; STATE_ONLY: only the state leaving the unit;
// NU: operands the weighted y is split into in the state's update (bf16).
template <typename T, typename OT, int E, bool FWD, bool STATE_ONLY, int NU>
__global__ __launch_bounds__(kThreads, 2) void walk_kernel(WalkArgs<T, OT> a) {
  using M = Lds<T, E>;
  __shared__ M s;
  constexpr int KS = E / 32, ET = E / 64, FN = kFT / 16, NS = M::kSplit;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, lg = lane >> 4;
  // tiles of one unit share x and y: they follow each other on one XCD (workgroups go round the 8 in turn)
  const int slot = blockIdx.x >> 3;
  const int64_t unit = (int64_t)(slot / a.nft) * 8 + (blockIdx.x & 7);
  if (unit >= a.units) return;
  const int f0 = (slot % a.nft) * kFT, ft_id = slot % a.nft;
  const int seg = (int)(unit % a.nseg);
  const int64_t bh = unit / a.nseg, b = bh / a.H, nbh = a.units / a.nseg;
  const int h = (int)(bh % a.H);
  const int nchunk = (int)((a.L + kC - 1) / kC);
  const int c_lo = seg * a.seg_chunks, c_hi = min(nchunk, c_lo + a.seg_chunks);
  const int64_t kv = (int64_t)a.E * a.F;

  // the state tile: wave w owns rows e = 16 (w ET + et) + 4 lg + r of columns f0 + 16 ft + li
  f32x4 S[ET][FN];
  const float* init = a.init ? a.init + (a.init_per_seg ? unit : bh) * kv : nullptr;
#pragma unroll
  for (int et = 0; et < ET; ++et)
#pragma unroll
    for (int ft = 0; ft < FN; ++ft)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int e = 16 * (wave * ET + et) + 4 * lg + r, f = f0 + 16 * ft + li;
        S[et][ft][r] = init && e < a.E && f < a.F ? init[(int64_t)e * a.se + (int64_t)f * a.sf] : 0.0f;
      }

  auto state_to_lds = [&]() {
#pragma unroll
    for (int et = 0; et < ET; ++et)
#pragma unroll
      for (int ft = 0; ft < FN; ++ft) {
        T* row = s.s[0] + (16 * ft + li) * M::kRow + 16 * (wave * ET + et) + 4 * lg;
        f32x4 rest = S[et][ft];
#pragma unroll
        for (int n = 0; n < NS; ++n) {
          T v[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            v[r] = from_f32<T>(rest[r]);
            rest[r] -= to_f32(v[r]);
          }
          __builtin_memcpy(__builtin_assume_aligned(row + n * kFT * M::kRow, 4 * sizeof(T)), v, sizeof(v));
        }
      }
  };

  // this thread's 4 x 8 pieces of y (E / 128 or half of one) and z
  constexpr int YC = E / 8, YN = (kC / 4) * YC, ZC = kFT / 8, ZN = (kC / 4) * ZC;
  constexpr int YP = (YN + kThreads - 1) / kThreads;
  Piece<T> py[YP], pz;
  auto fetch_chunk = [&](int c) {
    const int64_t t0 = (int64_t)c * kC;
#pragma unroll
    for (int p = 0; p < YP; ++p) {
      const int id = p * kThreads + threadIdx.x;
      if (id < YN) fetch(py[p], a.y, b, t0 + id / YC * 4, a.L, h, id % YC * 8, a.E);
    }
    if (threadIdx.x < ZN) fetch(pz, a.z, b, t0 + threadIdx.x / ZC * 4, a.L, h, f0 + threadIdx.x % ZC * 8, a.F);
  };
  Frag<T> x[KS];
  auto fetch_x = [&](int c) {
    const int64_t t = (int64_t)c * kC + 16 * wave + li;
    const T* p = a.x.row(b, t < a.L ? t : 0, h);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) load8(x[ks], p + 32 * ks + 8 * lg, t < a.L ? a.E - 32 * ks - 8 * lg : 0);
  };
  constexpr int kGateWave = FWD ? 0 : 3;  // the wave with the fewest score tiles

  double log_decay = 0.0;
  int c = FWD ? c_lo : c_hi - 1;
  if (c_lo < c_hi) {
    fetch_chunk(c);
    if (wave == kGateWave) gates<T, E, FWD>(s, 0, a, b, h, (int64_t)c * kC, lane);
  }
  if constexpr (!STATE_ONLY) state_to_lds();

  for (int n = 0; n < c_hi - c_lo; ++n, c += FWD ? 1 : -1) {
    const int buf = n & 1;
    if (FWD && !STATE_ONLY && a.anchors && c % a.anchor_chunks == 0) {
      float* to = a.anchors + (bh * a.nanchor + c / a.anchor_chunks) * kv;
#pragma unroll
      for (int et = 0; et < ET; ++et)
#pragma unroll
        for (int ft = 0; ft < FN; ++ft)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int e = 16 * (wave * ET + et) + 4 * lg + r, f = f0 + 16 * ft + li;
            if (e < a.E && f < a.F) to[(int64_t)e * a.se + (int64_t)f * a.sf] = S[et][ft][r];
          }
    }
#pragma unroll
    for (int p = 0; p < YP; ++p) {
      const int id = p * kThreads + threadIdx.x;
      if (id < YN) {
        if (!STATE_ONLY || !M::kBf) lds_rows(s.y, M::kRow, id / YC * 4, id % YC * 8, py[p]);
        lds_cols(s.yt, M::kCol, id / YC * 4, id % YC * 8, py[p]);
      }
    }
    if (threadIdx.x < ZN) {
      if constexpr (M::kBf)
        lds_cols(s.z, M::kCol, threadIdx.x / ZC * 4, threadIdx.x % ZC * 8, pz);
      else
        lds_rows(s.z, M::kZRow, threadIdx.x / ZC * 4, threadIdx.x % ZC * 8, pz);
    }
    if constexpr (!STATE_ONLY) fetch_x(c);
    __syncthreads();
    if (n + 1 < c_hi - c_lo) {
      fetch_chunk(c + (FWD ? 1 : -1));
      if (wave == kGateWave) gates<T, E, FWD>(s, buf ^ 1, a, b, h, (int64_t)(c + (FWD ? 1 : -1)) * kC, lane);
    }
    const float tot = FWD ? s.in[buf][kC - 1] : s.w[buf][kC - 1];  // the whole chunk's decay
    if constexpr (STATE_ONLY) log_decay += (double)s.hi[buf][kC - 1] + (double)s.lo[buf][kC - 1];

    if constexpr (!STATE_ONLY) {
      // scores, transposed: rows j = 16 jt + 4 lg + r, column i = 16 wave + li; P as operands over steps
      const int i = 16 * wave + li;
      const int64_t t = (int64_t)c * kC + i;
      const float gi_hi = s.hi[buf][i], gi_lo = s.lo[buf][i], in = s.in[buf][i];
      Frag<T> P[2][NS];
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        float p[8];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int jt = 2 * half + q;
          f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
          if (FWD ? jt <= wave : jt >= wave) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) acc = mma(lds_row(s.y + (16 * jt + li) * M::kRow + 32 * ks + 8 * lg), x[ks], acc);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int j = 16 * jt + 4 * lg + r;
            const float d = (gi_hi - s.hi[buf][j]) + (gi_lo - s.lo[buf][j]);
            const bool live = FWD ? j <= i : j >= i;
            p[4 * q + r] = live ? acc[r] * fast_exp2(FWD ? d : -d) : 0.0f;
          }
        }
        split<T, NS>(p, P[half]);
      }
      float dot = 0.0f;
#pragma unroll
      for (int ft = 0; ft < FN; ++ft) {
        f32x4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int m = 0; m < NS; ++m) acc = mma(lds_row(s.s[m] + (16 * ft + li) * M::kRow + 32 * ks + 8 * lg), x[ks], acc);
        acc *= in;
#pragma unroll
        for (int half = 0; half < 2; ++half)
          if (FWD ? 2 * half <= wave : 2 * half + 1 >= wave) {
            const Frag<T> zf = lds_col(s.z, M::kBf ? M::kCol : M::kZRow, 16 * ft + li, half, lg);
#pragma unroll
            for (int m = 0; m < NS; ++m) acc = mma(zf, P[half][m], acc);
          }
        const int f = f0 + 16 * ft + 4 * lg;
        if (t < a.L && f < a.F) {
          store4(a.out.row(b, t, h) + f, acc, a.F - f);
          if (a.dots) {
            const f32x4 u = load4(a.dot.row(b, t, h) + f, a.F - f);
#pragma unroll
            for (int r = 0; r < 4; ++r) dot = fmaf(acc[r], u[r], dot);
          }
        }
      }
      if (a.dots) {
        dot += __shfl_xor(dot, 16, kWave);
        dot += __shfl_xor(dot, 32, kWave);
        if (lg == 0 && t < a.L) a.dots[((int64_t)ft_id * nbh + bh) * a.L + t] = dot;
      }
    }

    // the state: S = tot S + sum_j (w_j y_j) z_j^T
    {
      Frag<T> zf[FN][2];
#pragma unroll
      for (int ft = 0; ft < FN; ++ft)
#pragma unroll
        for (int half = 0; half < 2; ++half) zf[ft][half] = lds_col(s.z, M::kBf ? M::kCol : M::kZRow, 16 * ft + li, half, lg);
#pragma unroll
      for (int et = 0; et < ET; ++et) {
#pragma unroll
        for (int ft = 0; ft < FN; ++ft) S[et][ft] *= tot;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const Frag<T> yf = lds_col(M::kBf ? s.yt : s.y, M::kBf ? M::kCol : M::kRow, 16 * (wave * ET + et) + li, half, lg);
          float wy[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) wy[e] = get(yf, e) * s.w[buf][32 * half + 16 * (e >> 2) + 4 * lg + (e & 3)];
          Frag<T> yw[M::kBf ? NU : 1];
          split<T, M::kBf ? NU : 1>(wy, yw);
#pragma unroll
          for (int ft = 0; ft < FN; ++ft)
#pragma unroll
            for (int m = 0; m < (M::kBf ? NU : 1); ++m) S[et][ft] = mma(yw[m], zf[ft][half], S[et][ft]);
        }
      }
    }
    if (!FWD && !STATE_ONLY && a.anchors && c % a.anchor_chunks == 0) {
      const float* from = a.anchors + (bh * a.nanchor + c / a.anchor_chunks) * kv;
      float d = 0.0f;
#pragma unroll
      for (int et = 0; et < ET; ++et)
#pragma unroll
        for (int ft = 0; ft < FN; ++ft)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int e = 16 * (wave * ET + et) + 4 * lg + r, f = f0 + 16 * ft + li;
            if (e < a.E && f < a.F) d = fmaf(from[(int64_t)e * a.se + (int64_t)f * a.sf], S[et][ft][r], d);
          }
      d = wave_sum(d);
      if (lane == 0) s.in[buf][16 * wave] = d;  // no other wave reads this step's weight
    }
    __syncthreads();
    if (!FWD && !STATE_ONLY && a.anchors && c % a.anchor_chunks == 0 && threadIdx.x == 0)
      a.anchor_dots[((int64_t)ft_id * nbh + bh) * a.nanchor + c / a.anchor_chunks] = (s.in[buf][0] + s.in[buf][16]) + (s.in[buf][32] + s.in[buf][48]);
    if constexpr (!STATE_ONLY) state_to_lds();
  }

  const bool end = STATE_ONLY || seg == (FWD ? a.nseg - 1 : 0);
  if (a.last && end) {
    float* to = a.last + (STATE_ONLY ? unit : bh) * kv;
#pragma unroll
    for (int et = 0; et < ET; ++et)
#pragma unroll
      for (int ft = 0; ft < FN; ++ft)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int e = 16 * (wave * ET + et) + 4 * lg + r, f = f0 + 16 * ft + li;
          if (e < a.E && f < a.F) to[(int64_t)e * a.se + (int64_t)f * a.sf] = S[et][ft][r];
        }
  }
  if constexpr (STATE_ONLY)
    if (threadIdx.x == 0 && ft_id == 0) a.seg_decay[unit] = log_decay;
}

// Segment states to entering states, in place: seg[n] becomes the state before segment n (after it, backwards).
__global__ __launch_bounds__(kThreads) void join_kernel(float* seg, const double* decay, const float* init, int nseg, int64_t kv, int64_t total,
                                                        int backward) {
  const int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (at >= total) return;
  const int64_t bh = at / kv, e = at % kv;
  float s = init ? init[at] : 0.0f;
  for (int n = 0; n < nseg; ++n) {
    const int64_t unit = bh * nseg + (backward ? nseg - 1 - n : n);
    const float own = seg[unit * kv + e];
    seg[unit * kv + e] = s;
    s = fmaf(fast_exp2((float)decay[unit]), s, own);
  }
}

// dg over one anchor's steps: the anchor's value, then the running sum of c - r before each step.
template <typename T>
__global__ __launch_bounds__(kThreads) void dgate_kernel(const float* r, const float* c, const float* anchor_dots, Seq<const T> g, Seq<T> dg, int H,
                                                         int64_t L, int64_t nbh, int nft, int anchor_steps, int nanchor) {
  __shared__ float part[4];
  const int64_t bh = blockIdx.x / nanchor;
  const int anchor = (int)(blockIdx.x % nanchor);
  const int64_t b = bh / H;
  const int h = (int)(bh % H);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float base = 0.0f;
  for (int f = 0; f < nft; ++f) base += anchor_dots[((int64_t)f * nbh + bh) * nanchor + anchor];
  for (int o = 0; o < anchor_steps; o += kThreads) {
    const int64_t t = (int64_t)anchor * anchor_steps + o + threadIdx.x;
    const bool in = o + (int)threadIdx.x < anchor_steps && t < L;
    float v = 0.0f;
    if (in)
      for (int f = 0; f < nft; ++f) {
        const int64_t at = ((int64_t)f * nbh + bh) * L + t;
        v += c[at] - r[at];
      }
    float sum = v;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
      const float up = __shfl_up(sum, d, kWave);
      if (lane >= d) sum += up;
    }
    if (lane == 63) part[wave] = sum;
    __syncthreads();
    float before = base;
    for (int w = 0; w < wave; ++w) before += part[w];
    if (in) {
      // where exp(g) is zero in fp32 the gradient is, whatever the sums' rounding left
      const bool none = to_f32(*g.row(b, t, h)) < -104.0f;
      *dg.row(b, t, h) = from_f32<T>(none ? 0.0f : before + (sum - v));
    }
    for (int w = 0; w < 4; ++w) base += part[w];
    __syncthreads();
  }
}

// Sums the heads that share a query or key head: [B, L, Hk, share, K] float32 to [B, L, Hk, K].
template <typename T>
__global__ __launch_bounds__(kThreads) void share_kernel(const float* in, T* out, int share, int K, int64_t total) {
  for (int64_t at = (int64_t)blockIdx.x * kThreads + threadIdx.x; at < total; at += (int64_t)gridDim.x * kThreads) {
    const float* p = in + at / K * share * K + at % K;
    float s = 0.0f;
    for (int r = 0; r < share; ++r) s += p[(int64_t)r * K];
    out[at] = from_f32<T>(s);
  }
}

// ------------------------------------------------------------------------------------------ step

struct StepArgs {
  const void *q, *k, *v, *g;
  int64_t qb, qh, kb, kh, vb, vh, gb, gh;
  float* state;
  void* o;
  int H, share, K, V, ntile;
};

// One step: a workgroup owns LANES 4-column pieces of one head's state; its threads split the K rows and
// each reads and writes its elements of the state once.
template <typename T, int LANES>
__global__ __launch_bounds__(kThreads) void step_kernel(StepArgs a) {
  constexpr int kRows = kThreads / LANES;
  __shared__ float qs[kStepMaxK], ks[kStepMaxK];
  __shared__ f32x4 part[kRows][LANES];
  const int tile = blockIdx.x % a.ntile;
  const int64_t bh = blockIdx.x / a.ntile, b = bh / a.H;
  const int h = (int)(bh % a.H), hk = h / a.share;
  const T* q = (const T*)a.q + b * a.qb + hk * a.qh;
  const T* k = (const T*)a.k + b * a.kb + hk * a.kh;
  for (int i = threadIdx.x; i < a.K; i += kThreads) {
    qs[i] = to_f32(q[i]);
    ks[i] = to_f32(k[i]);
  }
  const int lane = threadIdx.x % LANES, row = threadIdx.x / LANES;
  const int col = (tile * LANES + lane) * 4, n = a.V - col;
  const f32x4 v = n > 0 ? load4((const T*)a.v + b * a.vb + h * a.vh + col, n) : f32x4{0, 0, 0, 0};
  const float decay = fast_exp2(to_f32(((const T*)a.g)[b * a.gb + h * a.gh]) * kLog2e);
  __syncthreads();
  f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  if (n > 0) {
    float* st = a.state + bh * a.K * a.V + col;
#pragma unroll 8
    for (int i = row; i < a.K; i += kRows) {
      f32x4 s = load4(st + (int64_t)i * a.V, n);
      const float kk = ks[i], qq = qs[i];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[e] = fmaf(decay, s[e], kk * v[e]);
        sum[e] = fmaf(qq, s[e], sum[e]);
      }
      store4(st + (int64_t)i * a.V, s, n);
    }
  }
  part[row][lane] = sum;
  __syncthreads();
  if (row == 0 && n > 0) {
#pragma unroll
    for (int r = 1; r < kRows; ++r) sum += part[r][lane];
    store4((T*)a.o + bh * a.V + col, sum, n);
  }
}

// ------------------------------------------------------------------------------------------ host

struct Sizes {
  int64_t B, L, H, Hk, K, V;
};

int args_status(const Sizes& s, int dtype) {
  if (s.B < 0 || s.L < 0 || s.H < 1 || s.Hk < 1 || s.K < 1 || s.V < 1 || s.H % s.Hk != 0) return TSF_ERR_ARG;
  if (dtype != TSF_DTYPE_F32 && dtype != TSF_DTYPE_BF16) return TSF_ERR_ARG;
  if (s.K > kMaxWidth || s.V > kMaxWidth) return TSF_ERR_UNSUPPORTED;
  // workgroups of the largest launches: one a segment and tile, one an anchor, one per 256 state elements
  const int64_t chunks = (s.L + kC - 1) / kC, rows = s.B > 0 ? s.B : 1;
  if (s.H > (1 << 16) || s.L > ((int64_t)1 << 30) || rows > kMaxGrid / s.H) return TSF_ERR_UNSUPPORTED;
  const int64_t bh = rows * s.H;
  if (bh > kMaxGrid / 64 || bh * (chunks + 8) > kMaxGrid) return TSF_ERR_UNSUPPORTED;
  return TSF_OK;
}

int tiles(int64_t width) { return (int)((width + kFT - 1) / kFT); }

// Segments a row is cut into: enough workgroups for two on each CU, segments of four chunks at least.
int segments(const Sizes& s, int nft) {
  const int64_t chunks = (s.L + kC - 1) / kC, wgs = s.B * s.H * nft;
  int64_t n = wgs > 0 ? (2 * (int64_t)device_cus() + wgs - 1) / wgs : 1;
  if (n > chunks / 4) n = chunks / 4;
  if (n < 1) n = 1;
  const int64_t per = (chunks + n - 1) / n;
  return per > 0 ? (int)((chunks + per - 1) / per) : 1;
}

// Chunks between dg's anchors: an anchor's states cost 8 bytes a state element, the running sum's errors
// grow with the root of the distance; fp32 gates want the smaller error.
int anchor_chunks(int dtype) { return dtype == TSF_DTYPE_BF16 ? 16 : 4; }

int64_t align_up(int64_t n) { return (n + 255) & ~(int64_t)255; }

// Workspace: [segment states][segment decays] of the widest walk; backward also [r][c][anchors][anchor dots][dq, dk per head].
struct Space {
  int64_t seg, decay, r, c, anchors, anchor_dots, dq, dk, bytes;
};
Space space(const Sizes& s, int dtype, bool backward) {
  Space w = {};
  int64_t at = 0;
  const int64_t bh = s.B * s.H, kv = s.K * s.V;
  int nseg = segments(s, tiles(s.V));
  if (backward && segments(s, tiles(s.K)) > nseg) nseg = segments(s, tiles(s.K));
  auto take = [&](int64_t n) {
    const int64_t p = at;
    at += align_up(n);
    return p;
  };
  if (nseg > 1) {
    w.seg = take(bh * nseg * kv * 4);
    w.decay = take(bh * nseg * 8);
  }
  if (backward) {
    const int64_t chunks = (s.L + kC - 1) / kC, ac = anchor_chunks(dtype), na = (chunks + ac - 1) / ac, nk = tiles(s.K);
    w.r = take(nk * bh * s.L * 4);
    w.c = take(nk * bh * s.L * 4);
    w.anchors = take(bh * na * kv * 4);
    w.anchor_dots = take(nk * bh * na * 4);
    if (s.H != s.Hk) {
      w.dq = take(s.B * s.L * s.H * s.K * 4);
      w.dk = take(s.B * s.L * s.H * s.K * 4);
    }
  }
  w.bytes = at;
  return w;
}

template <typename T, typename OT, int E, bool FWD, int NU>
int walk_e(WalkArgs<T, OT> a, char* ws, const Space& sp, const float* init, float* last, hipStream_t stream) {
  const int64_t bh = a.units;
  const int64_t kv = (int64_t)a.E * a.F;
  a.units = bh * a.nseg;
  const unsigned grid = (unsigned)((a.units + 7) / 8 * 8 * a.nft);
  if (a.nseg > 1) {
    WalkArgs<T, OT> p = a;
    float* seg = (float*)(ws + sp.seg);
    double* decay = (double*)(ws + sp.decay);
    p.init = nullptr;
    p.last = seg;
    p.seg_decay = decay;
    walk_kernel<T, OT, E, FWD, true, NU><<<grid, kThreads, 0, stream>>>(p);
    const int64_t total = bh * kv;
    join_kernel<<<(unsigned)((total + kThreads - 1) / kThreads), kThreads, 0, stream>>>(seg, decay, init, a.nseg, kv, total, !FWD);
    a.init = seg;
    a.init_per_seg = 1;
  } else {
    a.init = init;
    a.init_per_seg = 0;
  }
  a.last = last;
  walk_kernel<T, OT, E, FWD, false, NU><<<grid, kThreads, 0, stream>>>(a);
  return tsf_launch_status();
}

// One walk. `init` and `last` are the row's states [row x head][K V]; a.units comes in as rows x heads.
template <typename T, typename OT, bool FWD, int NU>
int walk(WalkArgs<T, OT> a, const Sizes& s, char* ws, const Space& sp, const float* init, float* last, hipStream_t stream) {
  a.H = (int)s.H;
  a.L = s.L;
  a.units = s.B * s.H;
  a.nft = tiles(a.F);
  a.nseg = segments(s, a.nft);
  a.seg_chunks = (int)(((s.L + kC - 1) / kC + a.nseg - 1) / a.nseg);
  constexpr int N = sizeof(T) == 2 ? NU : 1;
  return a.E <= 64 ? walk_e<T, OT, 64, FWD, N>(a, ws, sp, init, last, stream) : walk_e<T, OT, 128, FWD, N>(a, ws, sp, init, last, stream);
}

template <typename T>
Seq<const T> seq_in(const void* p, const int64_t* st, int share) {
  return Seq<const T>{(const T*)p, st[0], st[1], st[2], share};
}

template <typename T>
int forward(const Sizes& s, const void* q, const void* k, const void* v, const void* g, const int64_t* st, const float* state, void* o, float* last,
            char* ws, const Space& sp, hipStream_t stream) {
  const int share = (int)(s.H / s.Hk);
  WalkArgs<T, T> a = {};
  a.x = seq_in<T>(q, st, share);
  a.y = seq_in<T>(k, st + 3, share);
  a.z = seq_in<T>(v, st + 6, 1);
  a.g = seq_in<T>(g, st + 9, 1);
  a.out = Seq<T>{(T*)o, s.L * s.H * s.V, s.H * s.V, s.V, 1};
  a.E = (int)s.K;
  a.F = (int)s.V;
  a.se = (int)s.V;
  a.sf = 1;
  return walk<T, T, true, 3>(a, s, ws, sp, state, last, stream);
}

// dq or dk: a walk over K's columns with V contracted, the dots of the gate's gradient beside it.
template <typename T, typename OT, bool FWD>
int walk_k(const Sizes& s, Seq<const T> x, Seq<const T> y, Seq<const T> z, Seq<const T> g, Seq<const T> dot, Seq<OT> out, float* dots, int dtype, char* ws, const Space& sp,
           const float* init, hipStream_t stream) {
  WalkArgs<T, OT> a = {};
  a.x = x;
  a.y = y;
  a.z = z;
  a.g = g;
  a.out = out;
  a.E = (int)s.V;
  a.F = (int)s.K;
  a.se = 1;
  a.sf = (int)s.V;
  a.dot = dot;
  a.dots = dots;
  a.anchors = (float*)(ws + sp.anchors);
  a.anchor_dots = (float*)(ws + sp.anchor_dots);
  a.anchor_chunks = anchor_chunks(dtype);
  a.nanchor = (int)(((s.L + kC - 1) / kC + a.anchor_chunks - 1) / a.anchor_chunks);
  return walk<T, OT, FWD, 2>(a, s, ws, sp, init, nullptr, stream);
}

template <typename T>
int backward(const Sizes& s, int dtype, const void* q, const void* k, const void* v, const void* g, const void* d_o, const int64_t* st, const float* state,
             const float* dlast, void* dq, void* dk, void* dv, void* dg, float* dstate, char* ws, const Space& sp, hipStream_t stream) {
  const int share = (int)(s.H / s.Hk);
  const Seq<const T> Q = seq_in<T>(q, st, share), Kk = seq_in<T>(k, st + 3, share), Vv = seq_in<T>(v, st + 6, 1), G = seq_in<T>(g, st + 9, 1),
                     DO = seq_in<T>(d_o, st + 12, 1);
  // dv, and the initial state's gradient
  {
    WalkArgs<T, T> a = {};
    a.x = Kk;
    a.y = Q;
    a.z = DO;
    a.g = G;
    a.out = Seq<T>{(T*)dv, s.L * s.H * s.V, s.H * s.V, s.V, 1};
    a.E = (int)s.K;
    a.F = (int)s.V;
    a.se = (int)s.V;
    a.sf = 1;
    const int rc = walk<T, T, false, 3>(a, s, ws, sp, dlast, dstate, stream);
    if (rc != TSF_OK) return rc;
  }
  if (s.L == 0) return TSF_OK;
  float *r = (float*)(ws + sp.r), *c = (float*)(ws + sp.c);
  int rc;
  if (share == 1) {
    const int64_t sl = s.H * s.K;
    rc = walk_k<T, T, true>(s, DO, Vv, Kk, G, Q, Seq<T>{(T*)dq, s.L * sl, sl, s.K, 1}, r, dtype, ws, sp, state, stream);
    if (rc != TSF_OK) return rc;
    rc = walk_k<T, T, false>(s, Vv, DO, Q, G, Kk, Seq<T>{(T*)dk, s.L * sl, sl, s.K, 1}, c, dtype, ws, sp, dlast, stream);
    if (rc != TSF_OK) return rc;
  } else {
    const int64_t sl = s.H * s.K, total = s.B * s.L * s.Hk * s.K;
    float *pq = (float*)(ws + sp.dq), *pk = (float*)(ws + sp.dk);
    rc = walk_k<T, float, true>(s, DO, Vv, Kk, G, Q, Seq<float>{pq, s.L * sl, sl, s.K, 1}, r, dtype, ws, sp, state, stream);
    if (rc != TSF_OK) return rc;
    rc = walk_k<T, float, false>(s, Vv, DO, Q, G, Kk, Seq<float>{pk, s.L * sl, sl, s.K, 1}, c, dtype, ws, sp, dlast, stream);
    if (rc != TSF_OK) return rc;
    const int64_t blocks = (total + kThreads - 1) / kThreads;
    const unsigned grid = (unsigned)(blocks < 65536 ? blocks : 65536);
    share_kernel<T><<<grid, kThreads, 0, stream>>>(pq, (T*)dq, share, (int)s.K, total);
    share_kernel<T><<<grid, kThreads, 0, stream>>>(pk, (T*)dk, share, (int)s.K, total);
  }
  const int ac = anchor_chunks(dtype);
  const int na = (int)(((s.L + kC - 1) / kC + ac - 1) / ac);
  dgate_kernel<T><<<(unsigned)(s.B * s.H * na), kThreads, 0, stream>>>(r, c, (const float*)(ws + sp.anchor_dots), G, Seq<T>{(T*)dg, s.L * s.H, s.H, 1, 1},
                                                                       (int)s.H, s.L, s.B * s.H, tiles(s.K), ac * kC, na);
  return tsf_launch_status();
}

}  // namespace

extern "C" {

int64_t tsfast_hip_gated_fwd_workspace_bytes(int64_t B, int64_t L, int64_t H, int64_t Hk, int64_t K, int64_t V, int dtype) {
  const Sizes s{B, L, H, Hk, K, V};
  return args_status(s, dtype) == TSF_OK ? space(s, dtype, false).bytes : -1;
}

int64_t tsfast_hip_gated_bwd_workspace_bytes(int64_t B, int64_t L, int64_t H, int64_t Hk, int64_t K, int64_t V, int dtype) {
  const Sizes s{B, L, H, Hk, K, V};
  return args_status(s, dtype) == TSF_OK ? space(s, dtype, true).bytes : -1;
}

int tsfast_hip_gated_fwd(int64_t B, int64_t L, int64_t H, int64_t Hk, int64_t K, int64_t V, int dtype, const void* q, const void* k, const void* v,
                         const void* g, const int64_t* strides, const float* state, void* o, float* state_last, void* workspace, int64_t workspace_bytes,
                         void* stream) {
  const Sizes s{B, L, H, Hk, K, V};
  const int rc = args_status(s, dtype);
  if (rc != TSF_OK) return rc;
  if (B == 0) return TSF_OK;
  if (!strides || !state_last || (L > 0 && (!q || !k || !v || !g || !o))) return TSF_ERR_ARG;
  const Space sp = space(s, dtype, false);
  if (sp.bytes > 0 && (!workspace || workspace_bytes < sp.bytes)) return TSF_ERR_WORKSPACE;
  return dtype == TSF_DTYPE_BF16 ? forward<bf16>(s, q, k, v, g, strides, state, o, state_last, (char*)workspace, sp, (hipStream_t)stream)
                                 : forward<float>(s, q, k, v, g, strides, state, o, state_last, (char*)workspace, sp, (hipStream_t)stream);
}

int tsfast_hip_gated_bwd(int64_t B, int64_t L, int64_t H, int64_t Hk, int64_t K, int64_t V, int dtype, const void* q, const void* k, const void* v,
                         const void* g, const void* grad_o, const int64_t* strides, const float* state, const float* grad_last, void* grad_q, void* grad_k,
                         void* grad_v, void* grad_g, float* grad_state, void* workspace, int64_t workspace_bytes, void* stream) {
  const Sizes s{B, L, H, Hk, K, V};
  const int rc = args_status(s, dtype);
  if (rc != TSF_OK) return rc;
  if (B == 0) return TSF_OK;
  if (!strides || (state && !grad_state)) return TSF_ERR_ARG;
  if (L > 0 && (!q || !k || !v || !g || !grad_o || !grad_q || !grad_k || !grad_v || !grad_g)) return TSF_ERR_ARG;
  const Space sp = space(s, dtype, true);
  if (sp.bytes > 0 && (!workspace || workspace_bytes < sp.bytes)) return TSF_ERR_WORKSPACE;
  return dtype == TSF_DTYPE_BF16 ? backward<bf16>(s, dtype, q, k, v, g, grad_o, strides, state, grad_last, grad_q, grad_k, grad_v, grad_g, grad_state,
                                                  (char*)workspace, sp, (hipStream_t)stream)
                                 : backward<float>(s, dtype, q, k, v, g, grad_o, strides, state, grad_last, grad_q, grad_k, grad_v, grad_g, grad_state,
                                                   (char*)workspace, sp, (hipStream_t)stream);
}

int tsfast_hip_gated_step(int64_t B, int64_t H, int64_t Hk, int64_t K, int64_t V, int dtype, const void* q, const void* k, const void* v, const void* g,
                          const int64_t* strides, float* state, void* o, void* stream) {
  if (B < 0 || H < 1 || Hk < 1 || K < 1 || V < 1 || H % Hk != 0 || (dtype != TSF_DTYPE_F32 && dtype != TSF_DTYPE_BF16)) return TSF_ERR_ARG;
  if (K > kStepMaxK || V > (1 << 20) || H > (1 << 20)) return TSF_ERR_UNSUPPORTED;
  if (B == 0) return TSF_OK;
  if (!q || !k || !v || !g || !strides || !state || !o) return TSF_ERR_ARG;
  StepArgs a{q, k, v, g, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], strides[6], strides[7], state, o,
             (int)H, (int)(H / Hk), (int)K, (int)V, 0};
  // wide pieces read whole rows of the state; narrow ones make more workgroups of a few heads
  const int64_t heads = B * H;
  const int lanes = V > 64 && heads >= 2 * (int64_t)device_cus() ? 32 : V > 16 && heads * ((V + 63) / 64) >= device_cus() ? 16 : 4;
  a.ntile = (int)((V + 4 * lanes - 1) / (4 * lanes));
  if (heads > kMaxGrid / a.ntile) return TSF_ERR_UNSUPPORTED;
  const unsigned grid = (unsigned)(heads * a.ntile);
  const hipStream_t st = (hipStream_t)stream;
  auto go = [&](auto lanes_c) {
    constexpr int N = decltype(lanes_c)::value;
    if (dtype == TSF_DTYPE_BF16)
      step_kernel<bf16, N><<<grid, kThreads, 0, st>>>(a);
    else
      step_kernel<float, N><<<grid, kThreads, 0, st>>>(a);
  };
  if (lanes == 32)
    go(std::integral_constant<int, 32>{});
  else if (lanes == 16)
    go(std::integral_constant<int, 16>{});
  else
    go(std::integral_constant<int, 4>{});
  return tsf_launch_status();
}

}  // extern "C"
