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
// so one kernel, walk_kernel, computes all four. A workgroup owns one head of one row and a run of 64-step chunks; the
// state stays in fp32 accumulator registers from the first chunk to the last. Per chunk
// the decayed scores of x and y within it (64 x 64, the causal half only) times z, x times the state before it, and the
// state's update are MFMA products; the decays come from exact differences of a float64 running sum, so that o, dq, dk and dv
// keep their accuracy for any g <= 0 down to -inf. Few rows are cut into segments: a walk of the state alone, a join of the segments' states, the
// walk proper; dk's walk takes its segments' states from dv's, and a training step's dq from o's.
//
// dg is a sum of terms that each carry their own decay from j < t to i >= t, so that it keeps its relative accuracy however
// strongly a head forgets, and a step that forgets all (g = -inf) parts the sequences of a packed row exactly. Within a chunk whose
// entering state is S and whose adjoint from beyond is T, with in_i and w_j the decays from its start and to its end,
//
//   dg_t = sum_{j < t <= i} D (q_i . k_j)(do_i . v_j) + sum_{i >= t} in_i q_i . (S do_i) + sum_{j < t} w_j k_j . (T v_j) + tot <S, T>.
//
// dq's walk has S and gives the first two, from its decayed scores and the part of dq that S makes, and leaves every chunk's S;
// dk's walk has T, adds the other two and writes dg. One head of 64 x 64, 1024 steps of constant g from -0.02 to -30, relative to the largest
// dg: 1e-7 to 1.2e-6 in fp32, 0.9e-3 to 2.5e-3 in bf16, one rounding of the result. (The shorter dg_{t+1} = dg_t - q_t . dq_t + k_t . dk_t
// is a difference of terms without exp(g_t): with it bf16 had 3e-2 at g = -8 and more than dg itself at -12, fp32 4e-2 there.) It costs
// a state a chunk, written and read: 2 x 805 MB at the size below, 13% of the training step.
//
// bf16 inputs are multiplied on the bf16 matrix cores. Products of inputs are exact there; what is fp32 (the decayed
// scores, the state, the decayed z of an update) goes in as a sum of two or three bf16 operands, because one alone (2^-9)
// would cost the outputs 1.4 times their own rounding, the fp32 state its type.
// fp32 inputs use the fp32 matrix cores.
//
// Time, 16 rows of 4096 steps, 12 heads of 128 x 128, bf16 (805 MB forward): 225 us for o's walk, 97 us for the
// segments' states before it and 34 for their join, 222 for dv's, 390 and 423 for dq's and dk's. No one unit bounds a chunk (4.7 us of a CU
// in o's walk): of it matrix products take 1.4 us, LDS 1.1 us and vector instructions about as much, waits for memory the rest; dq's and
// dk's add the chunks' states (64 KB each) and dq's the second score. Kept
// out, for they measured slower: the state in LDS as well (2 times), transposed copies of y and z in LDS instead of
// transposing reads (2 times, for their bank conflicts), eight waves of one column tile each (1.3 times),
// outputs stored from accumulators, 8 bytes a lane (1.35 times).
#include <math.h>

#include "common.h"
#include "tsfast_hip.h"

using namespace tsf;

namespace {

constexpr int kC = 64;                 // steps of a chunk
constexpr int kThreads = 256;          // of the small kernels
constexpr int kWaves = 4;              // of a walk: a workgroup takes all of its columns, so that nothing of x and y is done twice
constexpr int kMaxWidth = 128;         // of K and V
constexpr int kStepMaxK = 1024;        // of K in a single step
constexpr int64_t kMaxStep = 1 << 23;  // elements between the steps of a row
constexpr int kMaxGrid = (1 << 24) - 1;
// log2 decay that stands for all smaller ones, -inf among them: 2^-300 is zero in fp32, and sums of
// 64 such gates keep 1e-11 in their float64 sums
constexpr double kNoDecayLeft = -300.0;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4), may_alias));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2), may_alias));

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

TSF_DEV void put(Frag<bf16>& f, int e, float x) { f.v[e] = (__bf16)x; }
TSF_DEV void put(Frag<float>& f, int e, float x) {
  if (e < 4)
    f.lo[e & 3] = x;
  else
    f.hi[e & 3] = x;
}

// Two floats to bf16 pairs, rounded to nearest even (one instruction), and the pair back (two).
TSF_DEV uint32_t pack2(float a, float b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 v = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(uint32_t, v);
}
TSF_DEV float low(uint32_t p) { return __uint_as_float(p << 16); }
TSF_DEV float high(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

// 2 M values as the sum of N operands' words: bf16 carries 8 bits of each value's mantissa an operand.
template <int M, int N>
TSF_DEV void split_words(const float* x, uint32_t (&w)[N][M]) {
#pragma unroll
  for (int k = 0; k < M; ++k) {
    float a = x[2 * k], b = x[2 * k + 1];
#pragma unroll
    for (int n = 0; n < N; ++n) {
      w[n][k] = pack2(a, b);
      if (n + 1 < N) a -= low(w[n][k]), b -= high(w[n][k]);
    }
  }
}
// Eight values as the sum of N operands (fp32: as they are).
template <int N>
TSF_DEV void split(const float* x, Frag<bf16>* out) {
  uint32_t w[N][4];
  split_words<4, N>(x, w);
#pragma unroll
  for (int n = 0; n < N; ++n) __builtin_memcpy(&out[n].v, w[n], 16);
}
template <int N>
TSF_DEV void split(const float* x, Frag<float>* out) {
#pragma unroll
  for (int e = 0; e < 4; ++e) out->lo[e] = x[e], out->hi[e] = x[4 + e];
}
// The eight values of an operand, weighted.
TSF_DEV void weigh(const Frag<bf16>& f, f32x4 w0, f32x4 w1, float* v) {
  uint32_t p[4];
  __builtin_memcpy(p, &f.v, 16);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const f32x4& w = k < 2 ? w0 : w1;
    v[2 * k] = low(p[k]) * w[2 * (k & 1)];
    v[2 * k + 1] = high(p[k]) * w[2 * (k & 1) + 1];
  }
}
TSF_DEV void weigh(const Frag<float>& f, f32x4 w0, f32x4 w1, float* v) {
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = f.lo[e] * w0[e], v[4 + e] = f.hi[e] * w1[e];
}

// Eight consecutive values of a row of global memory at any alignment.
TSF_DEV void load8(Frag<bf16>& f, const bf16* p) { __builtin_memcpy(&f.v, p, 16); }
TSF_DEV void load8(Frag<float>& f, const float* p) {
  __builtin_memcpy(&f.lo, p, 16);
  __builtin_memcpy(&f.hi, p + 4, 16);
}
// The first n of a row's last values (any n: none, or all eight), zeros after, where there are eight values in a row: f was
// read so that it ends with the row.
TSF_DEV void fit(Frag<bf16>& f, int n) {
  const int s = n >= 8 ? 0 : n <= 0 ? 8 : 8 - n;  // places to move by
  u32x4 v = __builtin_bit_cast(u32x4, f.v);
  if (s & 1) v = u32x4{__builtin_amdgcn_alignbit(v[1], v[0], 16), __builtin_amdgcn_alignbit(v[2], v[1], 16), __builtin_amdgcn_alignbit(v[3], v[2], 16), v[3] >> 16};
  if (s & 2) v = u32x4{v[1], v[2], v[3], 0};
  if (s & 4) v = u32x4{v[2], v[3], 0, 0};
  if (s & 8) v = u32x4{0, 0, 0, 0};
  f.v = __builtin_bit_cast(bf16x8, v);
}
TSF_DEV void fit(Frag<float>& f, int n) {
  const int s = n >= 8 ? 0 : n <= 0 ? 8 : 8 - n;
  if (s & 1) f.lo = f32x4{f.lo[1], f.lo[2], f.lo[3], f.hi[0]}, f.hi = f32x4{f.hi[1], f.hi[2], f.hi[3], 0.0f};
  if (s & 2) f.lo = f32x4{f.lo[2], f.lo[3], f.hi[0], f.hi[1]}, f.hi = f32x4{f.hi[2], f.hi[3], 0.0f, 0.0f};
  if (s & 4) f.lo = f.hi, f.hi = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (s & 8) f.lo = f.hi = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
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
// Four consecutive values of a row of global memory at any alignment, zeros where there are fewer than n.
template <typename T>
TSF_DEV f32x4 load4(const T* p, int n) {
  f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  if (n >= 4) {
    T h[4];
    __builtin_memcpy(h, p, sizeof(h));
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = to_f32(h[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < n) v[e] = to_f32(p[e]);
  }
  return v;
}

// The first n of eight outputs to a row of global memory at any alignment; `rest` is what their rounding left.
TSF_DEV float value(const Frag<bf16>& o, int e) { return (float)o.v[e]; }
TSF_DEV float value(const Frag<float>& o, int e) { return e < 4 ? o.lo[e & 3] : o.hi[e & 3]; }
template <typename F>
TSF_DEV void store8(float* p, const F& o, const F& rest, int n) {
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = value(o, e) + value(rest, e);
  if (n >= 8) {
    __builtin_memcpy(p, v, 32);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = v[e];
  }
}
TSF_DEV void store8(bf16* p, const Frag<bf16>& o, const Frag<bf16>&, int n) {
  if (n >= 8) {
    __builtin_memcpy(p, &o.v, 16);
  } else {
    bf16 v[8];
    __builtin_memcpy(v, &o.v, 16);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) p[e] = v[e];
  }
}
// An element by a 32-bit index from an address that all lanes share.
template <typename T>
TSF_DEV T* at32(T* base, uint32_t idx) {
  return (T*)((char*)base + idx * (uint32_t)sizeof(T));
}

// A sequence tensor: strides in elements of the batch row, the step and the head; `share` heads of the
// state read one head of it. The innermost dimension is dense.
template <typename T>
struct Seq {
  T* p;
  int64_t sb, sl, sh;
  int share;
  TSF_DEV T* head(int64_t b, int h) const { return p + b * sb + (int64_t)(h / share) * sh; }
};

template <typename T, typename OT>
struct WalkArgs {
  Seq<const T> x, y, z, g;
  Seq<OT> out;
  int H, E, F;       // heads, columns of x and y, columns of z
  int64_t L, units;  // steps; rows x heads x segments
  int nseg, seg_chunks;
  int se, sf;             // strides of a caller's state's element (e, f)
  const float* init;      // state entering the row [row x head][K V], or null: zero
  const f32x4* seg_init;  // state entering each unit, where rows are cut
  float* last;            // state leaving the row
  f32x4* seg_last;        // STATE_ONLY: state leaving each unit
  double* seg_decay;      // STATE_ONLY: log2 of the unit's decay
  // of the gate's gradient (GATE): q for dq's walk, k for dk's; dg's part that dq's walk gives [row x head][L]; the states
  // entering the chunks [row x head][chunk]; both written forward, read backward
  Seq<const T> u;
  float* partial;
  f32x4* states;
  Seq<T> dg;
};

// 16 and 8 bytes of LDS as one access
template <int N>
TSF_DEV void lds_get(void* to, const char* p) {
  if constexpr (N == 16) {
    const u32x4 v = *(const u32x4*)p;
    __builtin_memcpy(to, &v, 16);
  } else {
    const u32x2 v = *(const u32x2*)p;
    __builtin_memcpy(to, &v, 8);
  }
}
template <int N>
TSF_DEV void lds_put(char* p, const void* from) {
  if constexpr (N == 16) {
    u32x4 v;
    __builtin_memcpy(&v, from, 16);
    *(u32x4*)p = v;
  } else {
    u32x2 v;
    __builtin_memcpy(&v, from, 8);
    *(u32x2*)p = v;
  }
}

// LDS arrays are rows of 16-byte units; unit u of row r stands at u ^ turn(r), so that 16 rows' same unit, and
// 16 columns of four rows, fall on different banks. x, y and the scores are operands over their columns: a
// unit pair (fp32) or a unit (bf16) holds one operand's 8 values, columns 32 s + 16 h + 4 lg + q in the order (h, q)
// for lane group lg, the order accumulators have them in. Rows are 128 bytes or more and a turn is below 16, so what
// selects s or t below is an exclusive or with a constant on a lane's own offset.
template <typename T, int COLS>
struct Rows {
  static constexpr bool kBf = sizeof(T) == 2;
  static constexpr int kBytes = COLS * (int)sizeof(T), kUnits = kBytes / 16, kHalf = 4 * (int)sizeof(T);
  alignas(16) char at[kC * kBytes];
  TSF_DEV static uint32_t turn(uint32_t r) {
    const uint32_t a = (r >> 2) & 3;
    if constexpr (!kBf) return r & 15;
    return (kUnits >= 16 ? (r & 3) << 2 : (r & 2) << 1) | ((a ^ (a << 1)) & 3);
  }
  // columns 8 m .. of row r (below 16), split into the two halves of operands; the offset of the first
  TSF_DEV static uint32_t piece(uint32_t r, uint32_t m) {
    if constexpr (kBf) return r * kBytes + ((((m >> 2) * 4 + (m & 1) * 2) ^ turn(r)) << 4) + ((m >> 1) & 1) * 8;
    return r * kBytes + (((2 * m) ^ turn(r)) << 4);
  }
  TSF_DEV void put_piece(uint32_t off, int row16, const Frag<T>& f) {
    char* p = at + row16 * 16 * kBytes;
    lds_put<kHalf>(p + off, &f);
    lds_put<kHalf>(p + (off ^ 16), (const char*)&f + kHalf);
  }
  // columns 8 m .. of row r (below 16) in their own order (z)
  TSF_DEV static uint32_t plain(uint32_t r, uint32_t m) { return kBf ? r * kBytes + ((m ^ turn(r)) << 4) : piece(r, m); }
  TSF_DEV void put_plain(uint32_t off, int row16, const Frag<T>& f) {
    if constexpr (kBf)
      lds_put<16>(at + row16 * 16 * kBytes + off, &f);
    else
      put_piece(off, row16, f);
  }
  TSF_DEV Frag<T> get_plain(uint32_t off, int row16) const {
    Frag<T> f;
    const char* p = at + row16 * 16 * kBytes;
    lds_get<16>(&f, p + off);
    if constexpr (!kBf) lds_get<16>(&f.hi, p + (off ^ 16));
    return f;
  }
  // four columns 16 tile + 4 lg .. of row 16 t + li, as accumulators have them, to plain places: the lane's offset, and the move
  TSF_DEV static uint32_t four_lane(uint32_t li, uint32_t lg) {
    return kBf ? li * kBytes + (((lg >> 1) ^ turn(li)) << 4) + 8 * (lg & 1) : li * kBytes + ((lg ^ turn(li)) << 4);
  }
  TSF_DEV void put_plain_four(uint32_t lane_off, int t, int tile, const void* f) {
    lds_put<kHalf>(at + t * 16 * kBytes + (lane_off ^ (tile << (kBf ? 5 : 6))), f);
  }
  TSF_DEV f32x4 get_plain_four(uint32_t lane_off, int t, int tile) const {
    T v[4];
    lds_get<kHalf>(v, at + t * 16 * kBytes + (lane_off ^ (tile << (kBf ? 5 : 6))));
    return f32x4{to_f32(v[0]), to_f32(v[1]), to_f32(v[2]), to_f32(v[3])};
  }
  // operands whose row is row 16 t + li, over columns 32 s ..: the lane's offset, and the operand
  TSF_DEV static uint32_t row_lane(uint32_t li, uint32_t lg) { return li * kBytes + ((lg ^ turn(li)) << 4); }
  TSF_DEV Frag<T> row(uint32_t lane_off, int t, int s) const {
    Frag<T> f;
    const char* p = at + t * 16 * kBytes;
    if constexpr (kBf) {
      lds_get<16>(&f, p + (lane_off ^ (s << 6)));
    } else {
      lds_get<16>(&f.lo, p + (lane_off ^ (s << 7)));
      lds_get<16>(&f.hi, p + (lane_off ^ (s << 7 | 64)));
    }
    return f;
  }
  // four columns 16 jt + 4 lg .. of row 16 t + li, as accumulators have them
  TSF_DEV void put_four(uint32_t lane_off, int t, int jt, const void* f) {
    char* p = at + t * 16 * kBytes;
    if constexpr (kBf)
      lds_put<8>(p + (lane_off ^ ((jt >> 1) << 6)) + 8 * (jt & 1), f);
    else
      lds_put<16>(p + (lane_off ^ (jt << 6)), f);
  }
  // operands whose row is column 16 t + li and whose contraction runs over rows (steps) 32 half ..; OPERAND: columns are in
  // operand order. bf16: the transposing read, in which lane li of a group of 16 points at 4 columns of row li / 4 and
  // receives its own column of the 4 rows.
  template <bool OPERAND>
  TSF_DEV static uint32_t col_lane(uint32_t li, uint32_t lg) {
    const uint32_t r = 4 * lg + (li >> 2), m = li & 3;
    if constexpr (kBf) return r * kBytes + (((OPERAND ? m : m >> 1) ^ turn(r)) << 4) + (OPERAND ? 0 : 8 * (m & 1));
    return 0;
  }
  template <bool OPERAND>
  TSF_DEV Frag<T> col(uint32_t lane_off, int t, int half, uint32_t li, uint32_t lg) const {
    Frag<T> f;
    if constexpr (kBf) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const char* p = at + (32 * half + 16 * h) * kBytes + (OPERAND ? (lane_off ^ ((t >> 1) << 6)) + 8 * (t & 1) : (lane_off ^ (t << 5)));
        const auto w = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(
                                                     __attribute__((address_space(3))) char*)const_cast<char*>(p)));
#pragma unroll
        for (int q = 0; q < 4; ++q) f.v[4 * h + q] = w[q];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t r = 4 * lg + (e & 3);
        put(f, e, *(const float*)(at + (32 * half + 16 * (e >> 2)) * kBytes + r * kBytes + (((4 * t + (li >> 2)) ^ turn(r)) << 4) + 4 * (li & 3)));
      }
    }
    return f;
  }
};

template <typename T, int E, int FT>
struct Lds {
  static constexpr int kSplit = sizeof(T) == 2 ? 2 : 1;  // operands the state and the scores are split into
  union {
    Rows<T, E> x;
    Rows<T, FT> u;  // GATE: q or k, once x has been used
    Rows<T, FT> o;  // the outputs on their way to memory, once x (and u) have been used
  };
  Rows<T, E> y;
  Rows<T, FT> z;
  union {
    Rows<T, kC> p[kSplit];  // decayed scores, row i
    Rows<T, FT> o_rest;     // what the outputs' rounding left (fp32 from bf16), once the scores have been used
  };
  alignas(16) float hi[2][kC], lo[2][kC], w[2][kC], in[2][kC];  // running log2 decay, weights into the state and out of it
};

// Sums of the gate's gradient on their way between waves.
struct GateLds {
  float dots[kWaves][kC];               // u_i . (x_i times the state) over a wave's columns
  float rows[6][16], cols[6][16];       // of the score tiles below the diagonal, by tile_slot: sums over j of row i, over i of column j
  float diag[kC];                       // the pairs within a diagonal tile
  float with[kWaves];                   // <entering state, state> over a wave's columns
};
TSF_DEV int tile_slot(int it, int jt) { return it * (it - 1) / 2 + jt; }

// Four values over the 16 lanes of a row (`li`), each summed over them: lane li has the sum of value (li >> 2) of all.
TSF_DEV float sum_lanes16(const float (&v)[4], int li) {
  const bool b3 = li & 8, b2 = li & 4;
  float a0 = b3 ? v[2] : v[0], a1 = b3 ? v[3] : v[1];
  a0 += __shfl_xor(b3 ? v[0] : v[2], 8, kWave);
  a1 += __shfl_xor(b3 ? v[1] : v[3], 8, kWave);
  float a = b2 ? a1 : a0;
  a += __shfl_xor(b2 ? a0 : a1, 4, kWave);
  a += __shfl_xor(a, 2, kWave);
  return a + __shfl_xor(a, 1, kWave);
}
// Four values over the four groups of lanes (`lg`), each summed over them: group lg has the sum of value lg of all.
TSF_DEV float sum_groups(const float (&v)[4], int lg) {
  const bool b1 = lg & 2, b0 = lg & 1;
  float a0 = b1 ? v[2] : v[0], a1 = b1 ? v[3] : v[1];
  a0 += __shfl_xor(b1 ? v[0] : v[2], 32, kWave);
  a1 += __shfl_xor(b1 ? v[1] : v[3], 32, kWave);
  return (b0 ? a1 : a0) + __shfl_xor(b0 ? a0 : a1, 16, kWave);
}
// Sums over the lanes from a lane on, and up to one, of every W lanes.
template <int W>
TSF_DEV float suffix_sum(float x, int lane) {
#pragma unroll
  for (int d = 1; d < W; d <<= 1) {
    const float v = __shfl_down(x, d, kWave);
    if ((lane & (W - 1)) + d < W) x += v;
  }
  return x;
}
template <int W>
TSF_DEV float prefix_before(float x, int lane) {
#pragma unroll
  for (int d = 1; d < W; d <<= 1) {
    const float v = __shfl_up(x, d, kWave);
    if ((lane & (W - 1)) >= d) x += v;
  }
  x = __shfl_up(x, 1, kWave);
  return (lane & (W - 1)) ? x : 0.0f;
}

// One tile of the pairs' terms p = D (q_i . k_j)(do_i . v_j), rows i = 16 it + li, columns j = 16 jt + 4 lg + r: what the sums over
// j < t <= i need of it.
TSF_DEV void put_pairs(GateLds& g, const float (&p)[4], int it, int jt, int li, int lg, int lane) {
  const int col = 4 * lg + (li >> 2);
  if (it != jt) {
    float row = (p[0] + p[1]) + (p[2] + p[3]);
    row += __shfl_xor(row, 16, kWave);
    row += __shfl_xor(row, 32, kWave);
    const float sum = sum_lanes16(p, li);
    const int at = tile_slot(it, jt);
    if (lg == 0) g.rows[at][li] = row;
    if ((li & 3) == 0) g.cols[at][col] = sum;
  } else {
    // row i's sum over j < t, for the t of the columns; of rows i >= t alone
    const float s1 = p[0] + p[1], s2 = s1 + p[2];
    float before = s2 + p[3];
    float v = __shfl_up(before, 16, kWave);
    if (lane >= 16) before += v;
    v = __shfl_up(before, 32, kWave);
    if (lane >= 32) before += v;
    before = __shfl_up(before, 16, kWave);
    if (lane < 16) before = 0.0f;
    const float r[4] = {li >= 4 * lg ? before : 0.0f, li >= 4 * lg + 1 ? before + p[0] : 0.0f, li >= 4 * lg + 2 ? before + s1 : 0.0f,
                        li >= 4 * lg + 3 ? before + s2 : 0.0f};
    const float sum = sum_lanes16(r, li);
    if ((li & 3) == 0) g.diag[16 * it + col] = sum;
  }
}
// One wave, lane t: the pairs' sum over j < t <= i of the whole chunk.
TSF_DEV float pair_sums(const GateLds& g, int li, int lg, int lane) {
  float a = 0.0f, b = 0.0f, m = 0.0f;  // tiles of t's rows, of its columns, and below and left of both
#pragma unroll
  for (int it = 1; it < 4; ++it)
#pragma unroll
    for (int jt = 0; jt < it; ++jt) {
      const float row = g.rows[tile_slot(it, jt)][li], col = g.cols[tile_slot(it, jt)][li];
      if (lg == it) a += row;
      if (lg == jt) b += col;
      if (lg > jt && lg < it) m += row;
    }
#pragma unroll
  for (int d = 8; d >= 1; d >>= 1) m += __shfl_xor(m, d, kWave);
  return g.diag[lane] + suffix_sum<16>(a, lane) + prefix_before<16>(b, lane) + m;
}

// Waves a SIMD holds of a walk: what LDS and a 512-register file allow.
template <typename T>
constexpr int walk_waves(int E, int FW) {
  return sizeof(T) == 2 || (E == 64 && FW == 1) ? 2 : 1;
}

// One wave: the chunk's running log2 decay as float pairs (differences are exact to float64 rounding), the
// weight of each step in the state leaving the chunk, and of the state entering it at each step.
template <bool FWD, typename S>
TSF_DEV void gates(S& s, int buf, float g, int lane) {
  const double x = (double)g * 1.4426950408889634;
  double G = x < kNoDecayLeft ? kNoDecayLeft : x;  // NaN stays
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

// Hides from the compiler that a value is the one of the last iteration.
template <typename V>
TSF_DEV void again(V& v) {
  asm volatile("" : "+v"(v));
}

TSF_DEV float wave_sum(float x) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) x += __shfl_xor(x, m, kWave);
  return x;
}

TSF_DEV f32x4 four(const float* p) {
  f32x4 v;
  lds_get<16>(&v, (const char*)p);
  return v;
}

// E: columns of x and y, padded; FW: 16-column tiles of z a wave owns; FWD: the direction in time;
// STATE_ONLY: only the state leaving the unit; GATE: the gate's gradient too (dq's and dk's walks).
//
// The weighted z of the state's update is split into three bf16 operands where the caller gets the state (2^-24), two where
// only results follow that are rounded to bf16 (2^-16).
//
// Wave w owns the state's columns 16 (w FW + fw) + li, all E rows of them: accumulators S[fw][et] hold rows 16 et + 4 lg + r, which
// two by two are operands as they stand. Per chunk: (1) x, y, z to LDS; (2) the ten live 16 x 16 score tiles, shared
// among the waves, decayed and split into LDS, and x times the state; (3) the scores times z, the outputs, the state's update. With
// GATE, u takes x's place before (3), for its products with x times the state and, in dq's walk, with z = k: the pairs' second score.
template <typename T, typename OT, int E, int FW, bool FWD, bool STATE_ONLY, bool GATE>
__global__ __launch_bounds__(64 * kWaves, walk_waves<T>(E, FW)) void walk_kernel(WalkArgs<T, OT> a) {
  constexpr int kThr = 64 * kWaves, FT = 16 * kWaves * FW, KS = E / 32, ET = E / 16, NS = Lds<T, E, FT>::kSplit, NU = sizeof(T) == 4 ? 1 : GATE ? 2 : 3;
  constexpr bool kRest = sizeof(T) == 2 && sizeof(OT) == 4;  // heads that share q and k, summed before they are rounded: outputs go to LDS in two parts
  constexpr bool kGate = GATE && !STATE_ONLY;
  __shared__ Lds<T, E, FT> s;
  __shared__ GateLds gs;
  int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // the same in all lanes, as the compiler now knows
  const int64_t unit = blockIdx.x;
  const int seg = (int)(unit % a.nseg);
  if constexpr (STATE_ONLY)
    if (seg == (FWD ? a.nseg - 1 : 0)) return;  // no segment enters with its state
  const int64_t bh = unit / a.nseg, b = bh / a.H;
  const int h = (int)(bh % a.H);
  const int nchunk = (int)((a.L + kC - 1) / kC);
  const int c_lo = seg * a.seg_chunks, chunks = min(nchunk, c_lo + a.seg_chunks) - c_lo;
  const T *xh = a.x.head(b, h), *yh = a.y.head(b, h), *zh = a.z.head(b, h), *gh = a.g.head(b, h);
  OT* const oh = STATE_ONLY ? nullptr : a.out.head(b, h);
  const T* const uh = kGate ? a.u.head(b, h) : nullptr;
  // the lane's places in the LDS arrays
  uint32_t row_off = Rows<T, E>::row_lane(li, lg), p_off = Rows<T, kC>::row_lane(li, lg);
  uint32_t ycol_off = Rows<T, E>::template col_lane<true>(li, lg), zcol_off = Rows<T, FT>::template col_lane<false>(li, lg), o_off = Rows<T, FT>::four_lane(li, lg);

  // The state. In the workspace a segment's state is f32x4 [et][thread], padding included; the caller's
  // are K V floats, (e, f) at e se + f sf.
  f32x4 S[FW][ET];
  const int64_t kv = (int64_t)a.E * a.F;
  auto each_state = [&](auto f) {  // value = f(index in a caller's state, value)
#pragma unroll
    for (int fw = 0; fw < FW; ++fw)
#pragma unroll
      for (int et = 0; et < ET; ++et)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int e = 16 * et + 4 * lg + r, col = 16 * (wave * FW + fw) + li;
          if (e < a.E && col < a.F) S[fw][et][r] = f((int64_t)e * a.se + (int64_t)col * a.sf, S[fw][et][r]);
        }
  };
  auto each_tile = [&](auto f) {  // f(index of a thread's f32x4 in a workspace state, S's)
#pragma unroll
    for (int fw = 0; fw < FW; ++fw)
#pragma unroll
      for (int et = 0; et < ET; ++et) f((fw * ET + et) * kThr + threadIdx.x, S[fw][et]);
  };
  constexpr int kTiles = FW * ET * kThr;
  each_tile([](int, f32x4& v) { v = f32x4{0.0f, 0.0f, 0.0f, 0.0f}; });
  if (a.seg_init) {
    const f32x4* from = a.seg_init + unit * kTiles;
    each_tile([&](int at, f32x4& v) { v = from[at]; });
  } else if (a.init) {
    const float* init = a.init + bh * kv;
    each_state([&](int64_t at, float) { return init[at]; });
  }

  // this thread's 8-column pieces of x, y and z on their way to LDS: one of every kRowsX (kRowsZ) rows
  constexpr int XC = E / 8, kRowsX = kThr / XC, XP = kC / kRowsX, ZC = FT / 8, kRowsZ = kThr / ZC, ZP = kC / kRowsZ;
  Frag<T> px[STATE_ONLY ? 1 : XP], py[XP], pz[ZP], pu[kGate ? ZP : 1];
  int xrow = threadIdx.x / XC, xcol = threadIdx.x % XC * 8, zrow = threadIdx.x / ZC, zcol = threadIdx.x % ZC * 8;
  uint32_t x_lds = Rows<T, E>::piece(xrow & 15, xcol / 8) + (xrow >> 4) * 16 * Rows<T, E>::kBytes;
  uint32_t z_lds = Rows<T, FT>::plain(zrow & 15, zcol / 8) + (zrow >> 4) * 16 * Rows<T, FT>::kBytes;
  // A piece that ends beyond its row is read so that it ends with it, a row beyond the last step is read as the last one; what does
  // not belong goes on the way to LDS. Rows of fewer than eight columns are read by elements then.
  const bool exact = a.E == E && a.F == FT, narrow_x = a.E < 8, narrow_z = a.F < 8;
  const uint32_t x_most = a.E - 8, z_most = a.F - 8;
  auto fetch_chunk = [&](int c) {
    const int64_t t0 = (int64_t)c * kC;
    const int last = (int)min((int64_t)kC, a.L - t0) - 1;
    const T *xb = xh + t0 * a.x.sl, *yb = yh + t0 * a.y.sl, *zb = zh + t0 * a.z.sl;  // the same for all lanes
    if (!narrow_x) {
      const uint32_t col = min((uint32_t)xcol, x_most);
#pragma unroll
      for (int p = 0; p < XP; ++p) {
        const uint32_t row = min(p * kRowsX + xrow, last);
        load8(py[p], at32(yb, row * (uint32_t)a.y.sl + col));
        if constexpr (!STATE_ONLY) load8(px[p], at32(xb, row * (uint32_t)a.x.sl + col));
      }
    }
    if (!narrow_z) {
      const uint32_t col = min((uint32_t)zcol, z_most);
#pragma unroll
      for (int p = 0; p < ZP; ++p) load8(pz[p], at32(zb, (uint32_t)min(p * kRowsZ + zrow, last) * (uint32_t)a.z.sl + col));
    }
  };
  auto by_elements = [&](Frag<T>& f, const T* row, int col, int n) {
#pragma unroll
    for (int e = 0; e < 8; ++e) put(f, e, e < n ? to_f32(row[col + e]) : 0.0f);
  };
  auto fit_chunk = [&](int64_t t0) {
    const int steps = (int)min((int64_t)kC, a.L - t0);
#pragma unroll
    for (int p = 0; p < XP; ++p) {
      const int row = p * kRowsX + xrow, n = row < steps ? a.E - xcol : 0;
      if (narrow_x) {
        by_elements(py[p], yh + (t0 + row) * a.y.sl, xcol, n);
        if constexpr (!STATE_ONLY) by_elements(px[p], xh + (t0 + row) * a.x.sl, xcol, n);
      } else {
        fit(py[p], n);
        if constexpr (!STATE_ONLY) fit(px[p], n);
      }
    }
#pragma unroll
    for (int p = 0; p < ZP; ++p) {
      const int row = p * kRowsZ + zrow, n = row < steps ? a.F - zcol : 0;
      if (narrow_z)
        by_elements(pz[p], zh + (t0 + row) * a.z.sl, zcol, n);
      else
        fit(pz[p], n);
    }
  };
  auto fetch_u = [&](int64_t t0) {  // for which x's place is free after the scores
    const int last = (int)min((int64_t)kC, a.L - t0) - 1;
    const T* ub = uh + t0 * a.u.sl;
    const uint32_t col = min((uint32_t)zcol, z_most);
    if (!narrow_z)
#pragma unroll
      for (int p = 0; p < ZP; ++p) load8(pu[p], at32(ub, (uint32_t)min(p * kRowsZ + zrow, last) * (uint32_t)a.u.sl + col));
  };
  constexpr int kGateWave = kWaves - 1;  // one of those with the fewest score tiles
  constexpr int kStep = FWD ? 1 : -1;
  int c = FWD ? c_lo : c_lo + chunks - 1;
  auto fetch_gate = [&](int n) {  // of the n-th chunk walked; a step that does not exist reads another
    const int64_t t = (int64_t)(FWD ? c_lo + n : c_lo + chunks - 1 - n) * kC + lane;
    return gh[(n < chunks && t < a.L ? t : 0) * a.g.sl];
  };
  auto gate_of = [&](int n, T g) { return (int64_t)(FWD ? c_lo + n : c_lo + chunks - 1 - n) * kC + lane < a.L ? to_f32(g) : 0.0f; };

  // The states entering the chunks: dq's walk leaves them, dk's multiplies them with its own, 32 rows at a time. Columns of padding
  // are left out, and any others read for them: their states are zero.
  const int ft_n = (a.F + 15) / 16;
  auto state_at = [&](int c, int fw) { return a.states + ((bh * nchunk + c) * ft_n + min(wave * FW + fw, ft_n - 1)) * (ET * 64); };  // [et][lane]
  auto put_state = [&](int c) {
#pragma unroll
    for (int fw = 0; fw < FW; ++fw)
      if (wave * FW + fw < ft_n)
#pragma unroll
        for (int et = 0; et < ET; ++et) *at32(state_at(c, fw), et * 64 + lane) = S[fw][et];
  };
  f32x4 other[kGate && !FWD ? 2 : 1][FW][2];
  auto fetch_state = [&](int c, int ks) {
#pragma unroll
    for (int fw = 0; fw < FW; ++fw)
#pragma unroll
      for (int e = 0; e < 2; ++e) other[ks & 1][fw][e] = *at32(state_at(c, fw), (2 * ks + e) * 64 + lane);
  };
  auto use_state = [&](float& sum, int ks) {
#pragma unroll
    for (int fw = 0; fw < FW; ++fw)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int r = 0; r < 4; ++r) sum = fmaf(other[ks & 1][fw][e][r], S[fw][2 * ks + e][r], sum);
    again(sum);  // formed here: beside its use it would hold the loads' registers until then
  };

  double log_decay = 0.0;
  T g_next = from_f32<T>(0.0f);
  if (chunks > 0) {
    fetch_chunk(c);
    if (wave == kGateWave) {
      gates<FWD>(s, 0, gate_of(0, fetch_gate(0)), lane);
      g_next = fetch_gate(1);
    }
  }
  for (int n = 0; n < chunks; ++n, c += kStep) {
    // what follows from these is formed again in each chunk: kept over the loop it would not fit the registers beside the state
    again(lane), again(li), again(lg), again(row_off), again(p_off), again(ycol_off), again(zcol_off), again(o_off), again(x_lds), again(z_lds);
    again(xrow), again(xcol), again(zrow), again(zcol);
    const int buf = n & 1;
    const int64_t t0 = (int64_t)c * kC;
    [[maybe_unused]] float with = 0.0f, part_dg = 0.0f;
    if constexpr (kGate) {
      fetch_u(t0);
      if (!FWD && wave == 0) part_dg = a.partial[bh * a.L + min(t0 + lane, a.L - 1)];
    }
    if (!exact || t0 + kC > a.L) fit_chunk(t0);
#pragma unroll
    for (int p = 0; p < XP; ++p) {
      s.y.put_piece(x_lds, p * kRowsX / 16, py[p]);
      if constexpr (!STATE_ONLY) s.x.put_piece(x_lds, p * kRowsX / 16, px[p]);
    }
#pragma unroll
    for (int p = 0; p < ZP; ++p) s.z.put_plain(z_lds, p * kRowsZ / 16, pz[p]);
    __syncthreads();
    if constexpr (kGate && !FWD) fetch_state(c, 0), fetch_state(c, 1);
    if (n + 1 < chunks) fetch_chunk(c + kStep);  // before any stores, which the loads would wait behind
    if constexpr (kGate && FWD) put_state(c);
    if constexpr (STATE_ONLY) log_decay += (double)s.hi[buf][kC - 1] + (double)s.lo[buf][kC - 1];

    f32x4 acc[FW][4];  // outputs, transposed: columns f + 16 fw of z by steps i = 16 it + li
    [[maybe_unused]] float scores[12 / kWaves][4];  // decayed, of this wave's tiles
    if constexpr (!STATE_ONLY) {
      // decayed scores, transposed in registers: rows j = 16 jt + 4 lg + r, column i = 16 it + li
#pragma unroll
      for (int k = 0; k < 12 / kWaves; ++k) {
        const int id = wave + kWaves * k;
        if (id >= 10) {  // the two beside the diagonal that operands reach into
          const int it = FWD ? 2 * (id - 10) : 3 - 2 * (id - 10), jt = FWD ? it + 1 : it - 1;
          const float none[4] = {};
#pragma unroll
          for (int m = 0; m < NS; ++m) s.p[m].put_four(p_off, it, jt, none);
        } else {
          const int big = id >= 6 ? 3 : id >= 3 ? 2 : id >= 1 ? 1 : 0, small = id - big * (big + 1) / 2;
          const int it = FWD ? big : 3 - big, jt = FWD ? small : 3 - small;
          f32x4 sc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) sc = mma(s.y.row(row_off, jt, ks), s.x.row(row_off, it, ks), sc);
          const f32x4 j_hi = four(s.hi[buf] + 16 * jt + 4 * lg), j_lo = four(s.lo[buf] + 16 * jt + 4 * lg);
          const float i_hi = s.hi[buf][16 * it + li], i_lo = s.lo[buf][16 * it + li];
          float part[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float d = (i_hi - j_hi[r]) + (i_lo - j_lo[r]);
            const int j = 4 * lg + r;
            const bool live = it != jt || (FWD ? j <= li : j >= li);
            part[r] = sc[r] * fast_exp2(live ? (FWD ? d : -d) : -INFINITY);
            if constexpr (kGate && FWD) scores[k][r] = part[r];
          }
          if constexpr (NS == 1) {
            s.p[0].put_four(p_off, it, jt, part);
          } else {
            uint32_t words[NS][2];
            split_words<2, NS>(part, words);
#pragma unroll
            for (int m = 0; m < NS; ++m) s.p[m].put_four(p_off, it, jt, words[m]);
          }
        }
      }
      // x times the state entering
#pragma unroll
      for (int fw = 0; fw < FW; ++fw)
#pragma unroll
        for (int it = 0; it < 4; ++it) acc[fw][it] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        if constexpr (kGate && !FWD) {
          use_state(with, ks);
          if (ks + 2 < KS) fetch_state(c, ks + 2);
        }
        Frag<T> sf[FW][NS];
#pragma unroll
        for (int fw = 0; fw < FW; ++fw) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = S[fw][2 * ks + (e >> 2)][e & 3];
          split<NS>(v, sf[fw]);
        }
#pragma unroll
        for (int it = 0; it < 4; ++it) {
          const Frag<T> xf = s.x.row(row_off, it, ks);
#pragma unroll
          for (int m = 0; m < NS; ++m)
#pragma unroll
            for (int fw = 0; fw < FW; ++fw) acc[fw][it] = mma(sf[fw][m], xf, acc[fw][it]);
        }
      }
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        const float in = s.in[buf][16 * it + li];
#pragma unroll
        for (int fw = 0; fw < FW; ++fw) acc[fw][it] *= in;
      }
    }
    if (wave == kGateWave && n + 1 < chunks) {
      gates<FWD>(s, buf ^ 1, gate_of(n + 1, g_next), lane);
      g_next = fetch_gate(n + 2);
    }
    if constexpr (!STATE_ONLY) __syncthreads();

    if constexpr (kGate) {
      if (!exact || t0 + kC > a.L)
#pragma unroll
        for (int p = 0; p < ZP; ++p) {
          const int64_t t = t0 + p * kRowsZ + zrow;
          const int n = t < a.L ? a.F - zcol : 0;
          if (narrow_z)
            by_elements(pu[p], uh + t * a.u.sl, zcol, n);
          else
            fit(pu[p], n);
        }
#pragma unroll
      for (int p = 0; p < ZP; ++p) s.u.put_plain(z_lds, p * kRowsZ / 16, pu[p]);
      __syncthreads();
      // u_i . (x_i times the state)
      float d[4];
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        d[it] = 0.0f;
#pragma unroll
        for (int fw = 0; fw < FW; ++fw) {
          const f32x4 u = s.u.get_plain_four(o_off, it, wave * FW + fw);
#pragma unroll
          for (int r = 0; r < 4; ++r) d[it] = fmaf(u[r], acc[fw][it][r], d[it]);
        }
      }
      gs.dots[wave][lane] = sum_groups(d, lg);
      if constexpr (FWD) {
        const uint32_t zrow_off = Rows<T, FT>::row_lane(li, lg);
#pragma unroll
        for (int k = 0; k < 12 / kWaves; ++k) {
          const int id = wave + kWaves * k;
          if (id < 10) {
            const int it = id >= 6 ? 3 : id >= 3 ? 2 : id >= 1 ? 1 : 0, jt = id - it * (it + 1) / 2;
            f32x4 sc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < FT / 32; ++ks) sc = mma(s.z.row(zrow_off, jt, ks), s.u.row(zrow_off, it, ks), sc);
            const float p[4] = {scores[k][0] * sc[0], scores[k][1] * sc[1], scores[k][2] * sc[2], scores[k][3] * sc[3]};
            put_pairs(gs, p, it, jt, li, lg, lane);
          }
        }
      } else {
        with = wave_sum(with);
        if (lane == 0) gs.with[wave] = with;
      }
    }
    if constexpr (!STATE_ONLY) {
      // the scores times z
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        Frag<T> zf[FW];
#pragma unroll
        for (int fw = 0; fw < FW; ++fw) zf[fw] = s.z.template col<false>(zcol_off, wave * FW + fw, half, li, lg);
#pragma unroll
        for (int it = 0; it < 4; ++it)
          if (FWD ? 2 * half <= it : 2 * half + 1 >= it)
#pragma unroll
            for (int m = 0; m < NS; ++m) {
              const Frag<T> pf = s.p[m].row(p_off, it, half);
#pragma unroll
              for (int fw = 0; fw < FW; ++fw) acc[fw][it] = mma(zf[fw], pf, acc[fw][it]);
            }
      }
      if constexpr (kGate) __syncthreads();  // the scores and u have been used
#pragma unroll
      for (int it = 0; it < 4; ++it)
#pragma unroll
        for (int fw = 0; fw < FW; ++fw) {
          if constexpr (sizeof(T) == 4) {
            s.o.put_plain_four(o_off, it, wave * FW + fw, &acc[fw][it]);
          } else {
            float v[4];
            __builtin_memcpy(v, &acc[fw][it], 16);
            uint32_t words[kRest ? 2 : 1][2];
            split_words<2, kRest ? 2 : 1>(v, words);
            s.o.put_plain_four(o_off, it, wave * FW + fw, words[0]);
            if constexpr (kRest) s.o_rest.put_plain_four(o_off, it, wave * FW + fw, words[1]);
          }
        }
    }
    // the state: S = tot S + sum_j y_j (w_j z_j)^T
    const float tot = FWD ? s.in[buf][kC - 1] : s.w[buf][kC - 1];  // the whole chunk's decay
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const f32x4 w0 = four(s.w[buf] + 32 * half + 4 * lg), w1 = four(s.w[buf] + 32 * half + 16 + 4 * lg);
      Frag<T> zw[FW][NU];
#pragma unroll
      for (int fw = 0; fw < FW; ++fw) {
        float v[8];
        weigh(s.z.template col<false>(zcol_off, wave * FW + fw, half, li, lg), w0, w1, v);
        split<NU>(v, zw[fw]);
      }
#pragma unroll
      for (int et = 0; et < ET; ++et) {
        const Frag<T> yf = s.y.template col<true>(ycol_off, et, half, li, lg);
#pragma unroll
        for (int fw = 0; fw < FW; ++fw)
          if (half == 0) S[fw][et] *= tot;
#pragma unroll
        for (int m = 0; m < NU; ++m)
#pragma unroll
          for (int fw = 0; fw < FW; ++fw) S[fw][et] = mma(yf, zw[fw][m], S[fw][et]);
      }
    }
    if constexpr (kGate) {
      if (wave == 0) {
        float d = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) d += gs.dots[w][lane];
        if constexpr (FWD) {
          d = suffix_sum<kC>(d, lane) + pair_sums(gs, li, lg, lane);
          if (t0 + lane < a.L) a.partial[bh * a.L + t0 + lane] = d;
        } else {
          float both = 0.0f;
#pragma unroll
          for (int w = 0; w < kWaves; ++w) both += gs.with[w];
          d = part_dg + prefix_before<kC>(d, lane) + tot * both;
          if (t0 + lane < a.L) a.dg.head(b, h)[(t0 + lane) * a.dg.sl] = from_f32<T>(d);
        }
      }
    }
    __syncthreads();
    if constexpr (!STATE_ONLY) {
      // the outputs leave in whole rows
      const int steps = (int)min((int64_t)kC, a.L - t0);
#pragma unroll
      for (int p = 0; p < ZP; ++p) {
        const int row = p * kRowsZ + zrow, n = row < steps ? a.F - zcol : 0;
        const Frag<T> o = s.o.get_plain(z_lds, p * kRowsZ / 16);
        Frag<T> rest = {};
        if constexpr (kRest) rest = s.o_rest.get_plain(z_lds, p * kRowsZ / 16);
        if (n > 0) store8(at32(oh + t0 * a.out.sl, row * (uint32_t)a.out.sl + zcol), o, rest, n);
      }
      __syncthreads();  // x's place is free again
    }
  }

  if constexpr (STATE_ONLY) {
    f32x4* to = a.seg_last + unit * kTiles;
    each_tile([&](int at, f32x4& v) { to[at] = v; });
    if (threadIdx.x == 0) a.seg_decay[unit] = log_decay;
  } else if (a.last && seg == (FWD ? a.nseg - 1 : 0)) {
    float* to = a.last + bh * kv;
    each_state([&](int64_t at, float v) { return to[at] = v; });
  }
}

// Segment states to entering states, in place: seg[n] becomes the state before segment n (after it, backwards). `threads`,
// `et` and `fw` are the walk's; a thread owns one f32x4 of a state. `turned`, if any, gets the same states as the walk over the other
// columns holds them (rows and columns exchanged; `et_turned` and `fw_turned` are that walk's).
constexpr int kJoinThreads = 64;  // few states make few workgroups
template <int N>
__global__ __launch_bounds__(kJoinThreads) void join_kernel(f32x4* seg, const double* decay, const float* init, int nseg, int threads, int et, int fw, int E, int F, int se,
                                                   int sf, int64_t total, int backward, float* turned, int et_turned, int fw_turned) {
  const int64_t at = (int64_t)blockIdx.x * kJoinThreads + threadIdx.x;
  if (at >= total) return;
  const int per = threads * et * fw;
  const int64_t bh = at / per;
  const int in = (int)(at % per), lane = in % threads & 63;
  const int e = in / threads % et * 16 + (lane >> 4) * 4, col = (in % threads / 64 * fw + in / threads / et) * 16 + (lane & 15);
  f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};
  if (init && col < F)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (e + r < E) s[r] = init[bh * E * F + (int64_t)(e + r) * se + (int64_t)col * sf];
  f32x4* p = seg + (bh * nseg + (backward ? nseg - 1 : 0)) * per + in;
  const double* d = decay + bh * nseg + (backward ? nseg - 1 : 0);
  const int64_t step = backward ? -(int64_t)per : per;
  // the place of (e, col), (e + 1, col) .. in a turned state: columns e .., row col
  const int tile = e / 16;
  float* t = turned ? turned + ((bh * nseg + (backward ? nseg - 1 : 0)) * per +
                                (tile % fw_turned * et_turned + col / 16) * threads + tile / fw_turned * 64 + (col % 16 / 4) * 16 + e % 16) * 4 + col % 4
                    : nullptr;
  // several segments' loads at a time, as each would otherwise wait for the last one's store (128 segments: 40 us, so 15)
  for (int n0 = 0; n0 < nseg; n0 += N) {
    f32x4 own[N];
    float keep[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const int n = min(n0 + k, nseg - 2);  // nothing follows the last one, and its own state was not formed
      own[k] = p[n * step];
      keep[k] = (float)d[backward ? -n : n];
    }
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (n0 + k < nseg) {
        p[(n0 + k) * step] = s;
        if (t)
#pragma unroll
          for (int r = 0; r < 4; ++r) t[(n0 + k) * step * 4 + r * 4] = s[r];
        s = fast_exp2(keep[k]) * s + own[k];
      }
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

// One step: a workgroup owns 64 columns of one head's state, 16 threads a row of them and 16 rows at a time; each
// thread reads and writes its elements of the state once, in 16-byte pieces at any alignment, and HBM bounds it. For 256
// rows of 12 heads of 128 x 128: 60 us, 403 MB. Tiles of 16 and 128 columns took 108 and 60 us there, 11.5 and 7.4 against
// 6.6 us for 16 rows, 4.0 and 4.0 against 3.4 us for one row of 4 heads of 64 x 64.
constexpr int kStepLanes = 16, kStepRows = kThreads / kStepLanes;
template <typename T>
__global__ __launch_bounds__(kThreads) void step_kernel(StepArgs a) {
  __shared__ float qs[kStepMaxK], ks[kStepMaxK];
  __shared__ f32x4 part[kStepRows][kStepLanes];
  const int tile = blockIdx.x % a.ntile;
  const int64_t bh = blockIdx.x / a.ntile, b = bh / a.H;
  const int h = (int)(bh % a.H), hk = h / a.share;
  const T* q = (const T*)a.q + b * a.qb + hk * a.qh;
  const T* k = (const T*)a.k + b * a.kb + hk * a.kh;
  for (int i = threadIdx.x; i < a.K; i += kThreads) {
    qs[i] = to_f32(q[i]);
    ks[i] = to_f32(k[i]);
  }
  const int lane = threadIdx.x % kStepLanes, row = threadIdx.x / kStepLanes;
  const int col = (tile * kStepLanes + lane) * 4, n = a.V - col;
  const f32x4 v = n > 0 ? load4((const T*)a.v + b * a.vb + h * a.vh + col, n) : f32x4{0, 0, 0, 0};
  const float decay = fast_exp2(to_f32(((const T*)a.g)[b * a.gb + h * a.gh]) * kLog2e);
  __syncthreads();
  f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  if (n > 0) {
    float* st = a.state + bh * a.K * a.V + col;
#pragma unroll 8
    for (int i = row; i < a.K; i += kStepRows) {
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
    for (int r = 1; r < kStepRows; ++r) sum += part[r][lane];
    store4((T*)a.o + bh * a.V + col, sum, n);
  }
}

// ------------------------------------------------------------------------------------------ host

struct Sizes {
  int64_t B, L, H, Hk, K, V;
};

// Steps of a chunk are reached by 32-bit byte offsets from its first; a single one may be at any distance from none.
bool steps_fit(const int64_t* strides, int tensors, int64_t L) {
  if (L <= 1) return true;
  for (int i = 0; i < tensors; ++i)
    if (strides[3 * i + 1] < 0 || strides[3 * i + 1] > kMaxStep) return false;
  return true;
}

int args_status(const Sizes& s, int dtype) {
  if (s.B < 0 || s.L < 0 || s.H < 1 || s.Hk < 1 || s.K < 1 || s.V < 1 || s.H % s.Hk != 0) return TSF_ERR_ARG;
  if (dtype != TSF_DTYPE_F32 && dtype != TSF_DTYPE_BF16) return TSF_ERR_ARG;
  if (s.K > kMaxWidth || s.V > kMaxWidth) return TSF_ERR_UNSUPPORTED;
  // workgroups of the largest launches: one a segment, one per 64 pieces of a state
  const int64_t chunks = (s.L + kC - 1) / kC, rows = s.B > 0 ? s.B : 1;
  if (s.H > (1 << 16) || s.L > ((int64_t)1 << 30) || rows > kMaxGrid / s.H) return TSF_ERR_UNSUPPORTED;
  const int64_t bh = rows * s.H;
  if (bh > kMaxGrid / 64 || bh * (chunks + 8) > kMaxGrid) return TSF_ERR_UNSUPPORTED;
  return TSF_OK;
}

int64_t padded_state(int64_t E, int64_t F) { return (E <= 64 ? 64 : 128) * (F <= 64 ? 64 : 128); }

// Segments a row is cut into: the number with the least time, in chunks walked one after the other, of one and those that
// fill every CU once or twice (a workgroup more, and the whole chip waits for another round: where two fitted a CU, 86 instead of 85
// segments of 6 rows took twice the time). A cut row's chunks are walked for the states too, at 0.45 times a chunk's time, and the states
// go to memory and back five times. Measured, training: 192 rows of 4096 steps, 128 x 128, bf16: whole 1999 us, 2 segments 1656, 5: 1537;
// 288 rows, 64 x 64: 1195, 972, 912; 192 rows of 2048, 64 x 64, fp32: 1032, 902, 826.
// Four chunks a segment at least. It is right for short bf16 rows (forward, 4 heads of 448 steps, 64 x 64: whole 23 us, in 4: 26) and for
// windows (128 rows of 512 steps, fp32, training: in 2, as they are, 192 us; 4: 188; 8: 209), and too high for few rows of slower chunks
// (forward, 4 heads, 512 steps of 64 x 64, fp32: in 2 43 us, 4: 27, 8: 26; 2048 of 128 x 128, bf16: in 8 44 us, 16: 32, 32: 30; training,
// 30 rows of 3001 of 48 x 80, bf16: in 10 234 us, 16: 188, 32: 215).
int segments(const Sizes& s, int dtype) {
  const int64_t chunks = (s.L + kC - 1) / kC, rows = s.B * s.H;
  const bool narrow = s.K <= 64 && s.V <= 64;
  const int64_t slots = (int64_t)device_cus() * (dtype == TSF_DTYPE_BF16 ? (narrow ? 3 : 2) : narrow ? 2 : 1);  // by their LDS
  if (rows < 1 || chunks < 8) return 1;
  double least = (double)((rows + slots - 1) / slots * chunks);
  int64_t best = 1;
  for (int64_t rounds = 1; rounds <= 2; ++rounds) {
    int64_t n = rounds * slots / rows;
    if (n > chunks / 4) n = chunks / 4;
    if (n < 2) continue;
    const int64_t per = (chunks + n - 1) / n;
    n = (chunks + per - 1) / per;
    const double time = (double)((rows * n + slots - 1) / slots * per) + 0.45 * (double)((rows * (n - 1) + slots - 1) / slots * per) +
                        1.2e-7 * (double)(padded_state(s.K, s.V) * 4 * rows * n);
    if (time < least) least = time, best = n;
  }
  return (int)best;
}

// Bytes of a chunk's state as dq's walk leaves it for dk's.
int64_t chunk_state(int64_t K, int64_t V) { return (K + 15) / 16 * 64 * (V <= 64 ? 64 : 128); }

int64_t align_up(int64_t n) { return (n + 255) & ~(int64_t)255; }

// Workspace: [segment states][segment decays]; backward also [segment states, turned][part of dg][chunks' states][dq, dk per head].
struct Space {
  int64_t seg, decay, turned, partial, states, dq, dk, bytes;
};
Space space(const Sizes& s, int dtype, bool backward) {
  Space w = {};
  int64_t at = 0;
  const int64_t bh = s.B * s.H, state = padded_state(s.K, s.V) * 4, nseg = segments(s, dtype);
  auto take = [&](int64_t n) {
    const int64_t p = at;
    at += align_up(n);
    return p;
  };
  if (nseg > 1) {
    w.seg = take(bh * nseg * state);
    w.decay = take(bh * nseg * 8);
    if (backward) w.turned = take(bh * nseg * state);
  }
  if (backward) {
    w.partial = take(bh * s.L * 4);
    w.states = take(bh * ((s.L + kC - 1) / kC) * chunk_state(s.K, s.V));
    if (s.H != s.Hk) {
      w.dq = take(s.B * s.L * s.H * s.K * 4);
      w.dk = take(s.B * s.L * s.H * s.K * 4);
    }
  }
  w.bytes = at;
  return w;
}

// One walk, cut rows' segment states first, unless `entering` has them. o's and dq's walks, and dv's and dk's, have the same
// states between segments with rows and columns exchanged: o's and dv's leave them in `turned` for the other (16 rows of 4096
// steps, 12 heads of 128 x 128, bf16: a state-only walk of 97 us and a join of 34 less each, for 63 MB that o's keeps).
template <typename T, typename OT, int E, int FW, bool FWD, bool GATE>
int walk_e(WalkArgs<T, OT> a, char* ws, const Space& sp, const float* init, float* last, const void* entering, void* turned,
           hipStream_t stream) {
  const int64_t bh = a.units;
  a.units = bh * a.nseg;
  if (a.nseg == 1) {
    a.init = init;
  } else if (entering || (!FWD && GATE)) {  // dk's always has them
    a.seg_init = (const f32x4*)entering;
  } else if constexpr (FWD || !GATE) {
    WalkArgs<T, OT> p = a;
    f32x4* seg = (f32x4*)(ws + sp.seg);
    p.seg_last = seg;
    p.seg_decay = (double*)(ws + sp.decay);
    walk_kernel<T, OT, E, FW, FWD, true, GATE><<<(unsigned)a.units, 64 * kWaves, 0, stream>>>(p);
    const int64_t total = bh * E / 16 * 64 * kWaves * FW;
    const auto join = a.nseg <= 4 ? join_kernel<4> : join_kernel<16>;
    join<<<(unsigned)((total + kJoinThreads - 1) / kJoinThreads), kJoinThreads, 0, stream>>>(seg, p.seg_decay, init, a.nseg, 64 * kWaves, E / 16, FW, a.E, a.F,
                                                                                            a.se, a.sf, total, !FWD, (float*)turned, FW * kWaves,
                                                                                            E / 16 / kWaves);
    a.seg_init = seg;
  }
  a.last = last;
  walk_kernel<T, OT, E, FW, FWD, false, GATE><<<(unsigned)a.units, 64 * kWaves, 0, stream>>>(a);
  return tsf_launch_status();
}

// One walk. `init` and `last` are the row's states [row x head][K V].
template <typename T, typename OT, bool FWD, bool GATE>
int walk(WalkArgs<T, OT> a, const Sizes& s, char* ws, const Space& sp, const float* init, float* last, const void* entering, void* turned,
         hipStream_t stream) {
  a.H = (int)s.H;
  a.L = s.L;
  a.units = s.B * s.H;
  a.nseg = segments(s, sizeof(T) == 2 ? TSF_DTYPE_BF16 : TSF_DTYPE_F32);
  a.seg_chunks = (int)(((s.L + kC - 1) / kC + a.nseg - 1) / a.nseg);
  const auto run = a.F <= 64 ? (a.E <= 64 ? walk_e<T, OT, 64, 1, FWD, GATE> : walk_e<T, OT, 128, 1, FWD, GATE>)
                             : (a.E <= 64 ? walk_e<T, OT, 64, 2, FWD, GATE> : walk_e<T, OT, 128, 2, FWD, GATE>);
  return run(a, ws, sp, init, last, entering, turned, stream);
}

template <typename T>
Seq<const T> seq_in(const void* p, const int64_t* st, int share) {
  return Seq<const T>{(const T*)p, st[0], st[1], st[2], share};
}

template <typename T>
int forward(const Sizes& s, const void* q, const void* k, const void* v, const void* g, const int64_t* st, const float* state, void* o, float* last,
            void* kept, char* ws, const Space& sp, hipStream_t stream) {
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
  return walk<T, T, true, false>(a, s, ws, sp, state, last, nullptr, kept, stream);
}

// dq or dk: a walk over K's columns with V contracted, the gate's gradient beside it.
template <typename T, typename OT, bool FWD>
int walk_k(const Sizes& s, Seq<const T> x, Seq<const T> y, Seq<const T> z, Seq<const T> g, Seq<const T> u, Seq<OT> out, void* dg, char* ws, const Space& sp,
           const float* init, const void* entering, hipStream_t stream) {
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
  a.u = u;
  a.partial = (float*)(ws + sp.partial);
  a.states = (f32x4*)(ws + sp.states);
  a.dg = Seq<T>{(T*)dg, s.L * s.H, s.H, 1, 1};
  return walk<T, OT, FWD, true>(a, s, ws, sp, init, nullptr, entering, nullptr, stream);
}

template <typename T>
int backward(const Sizes& s, const void* q, const void* k, const void* v, const void* g, const void* d_o, const int64_t* st, const float* state,
             const float* dlast, void* dq, void* dk, void* dv, void* dg, float* dstate, const void* kept, char* ws, const Space& sp,
             hipStream_t stream) {
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
    const int rc = walk<T, T, false, false>(a, s, ws, sp, dlast, dstate, nullptr, ws + sp.turned, stream);
    if (rc != TSF_OK) return rc;
  }
  if (s.L == 0) return TSF_OK;
  int rc;
  if (share == 1) {
    const int64_t sl = s.H * s.K;
    rc = walk_k<T, T, true>(s, DO, Vv, Kk, G, Q, Seq<T>{(T*)dq, s.L * sl, sl, s.K, 1}, dg, ws, sp, state, kept, stream);
    if (rc != TSF_OK) return rc;
    rc = walk_k<T, T, false>(s, Vv, DO, Q, G, Kk, Seq<T>{(T*)dk, s.L * sl, sl, s.K, 1}, dg, ws, sp, dlast, ws + sp.turned, stream);
    if (rc != TSF_OK) return rc;
  } else {
    const int64_t sl = s.H * s.K, total = s.B * s.L * s.Hk * s.K;
    float *pq = (float*)(ws + sp.dq), *pk = (float*)(ws + sp.dk);
    rc = walk_k<T, float, true>(s, DO, Vv, Kk, G, Q, Seq<float>{pq, s.L * sl, sl, s.K, 1}, dg, ws, sp, state, kept, stream);
    if (rc != TSF_OK) return rc;
    rc = walk_k<T, float, false>(s, Vv, DO, Q, G, Kk, Seq<float>{pk, s.L * sl, sl, s.K, 1}, dg, ws, sp, dlast, ws + sp.turned, stream);
    if (rc != TSF_OK) return rc;
    const int64_t blocks = (total + kThreads - 1) / kThreads;
    const unsigned grid = (unsigned)(blocks < 65536 ? blocks : 65536);
    share_kernel<T><<<grid, kThreads, 0, stream>>>(pq, (T*)dq, share, (int)s.K, total);
    share_kernel<T><<<grid, kThreads, 0, stream>>>(pk, (T*)dk, share, (int)s.K, total);
  }
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

// States between segments that the backward can take from the forward.
int64_t tsfast_hip_gated_kept_bytes(int64_t B, int64_t L, int64_t H, int64_t Hk, int64_t K, int64_t V, int dtype) {
  const Sizes s{B, L, H, Hk, K, V};
  if (args_status(s, dtype) != TSF_OK) return -1;
  const int64_t nseg = segments(s, dtype);
  return nseg > 1 ? B * H * nseg * padded_state(K, V) * 4 : 0;
}

int tsfast_hip_gated_fwd_train(int64_t B, int64_t L, int64_t H, int64_t Hk, int64_t K, int64_t V, int dtype, const void* q, const void* k, const void* v,
                               const void* g, const int64_t* strides, const float* state, void* o, float* state_last, void* kept, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  const Sizes s{B, L, H, Hk, K, V};
  const int rc = args_status(s, dtype);
  if (rc != TSF_OK) return rc;
  if (B == 0) return TSF_OK;
  if (!strides || !state_last || (L > 0 && (!q || !k || !v || !g || !o))) return TSF_ERR_ARG;
  if (!steps_fit(strides, 3, L)) return TSF_ERR_UNSUPPORTED;
  const Space sp = space(s, dtype, false);
  if (sp.bytes > 0 && (!workspace || workspace_bytes < sp.bytes)) return TSF_ERR_WORKSPACE;
  return dtype == TSF_DTYPE_BF16 ? forward<bf16>(s, q, k, v, g, strides, state, o, state_last, kept, (char*)workspace, sp, (hipStream_t)stream)
                                 : forward<float>(s, q, k, v, g, strides, state, o, state_last, kept, (char*)workspace, sp, (hipStream_t)stream);
}

int tsfast_hip_gated_fwd(int64_t B, int64_t L, int64_t H, int64_t Hk, int64_t K, int64_t V, int dtype, const void* q, const void* k, const void* v,
                         const void* g, const int64_t* strides, const float* state, void* o, float* state_last, void* workspace, int64_t workspace_bytes,
                         void* stream) {
  return tsfast_hip_gated_fwd_train(B, L, H, Hk, K, V, dtype, q, k, v, g, strides, state, o, state_last, nullptr, workspace, workspace_bytes, stream);
}

int tsfast_hip_gated_bwd_train(int64_t B, int64_t L, int64_t H, int64_t Hk, int64_t K, int64_t V, int dtype, const void* q, const void* k, const void* v,
                         const void* g, const void* grad_o, const int64_t* strides, const float* state, const float* grad_last, void* grad_q, void* grad_k,
                         void* grad_v, void* grad_g, float* grad_state, const void* kept, void* workspace, int64_t workspace_bytes, void* stream) {
  const Sizes s{B, L, H, Hk, K, V};
  const int rc = args_status(s, dtype);
  if (rc != TSF_OK) return rc;
  if (B == 0) return TSF_OK;
  if (!strides || (state && !grad_state)) return TSF_ERR_ARG;
  if (L > 0 && (!q || !k || !v || !g || !grad_o || !grad_q || !grad_k || !grad_v || !grad_g)) return TSF_ERR_ARG;
  if (!steps_fit(strides, 3, L) || !steps_fit(strides + 12, 1, L)) return TSF_ERR_UNSUPPORTED;
  const Space sp = space(s, dtype, true);
  if (sp.bytes > 0 && (!workspace || workspace_bytes < sp.bytes)) return TSF_ERR_WORKSPACE;
  return dtype == TSF_DTYPE_BF16 ? backward<bf16>(s, q, k, v, g, grad_o, strides, state, grad_last, grad_q, grad_k, grad_v, grad_g, grad_state, kept,
                                                  (char*)workspace, sp, (hipStream_t)stream)
                                 : backward<float>(s, q, k, v, g, grad_o, strides, state, grad_last, grad_q, grad_k, grad_v, grad_g, grad_state, kept,
                                                   (char*)workspace, sp, (hipStream_t)stream);
}

int tsfast_hip_gated_bwd(int64_t B, int64_t L, int64_t H, int64_t Hk, int64_t K, int64_t V, int dtype, const void* q, const void* k, const void* v,
                         const void* g, const void* grad_o, const int64_t* strides, const float* state, const float* grad_last, void* grad_q, void* grad_k,
                         void* grad_v, void* grad_g, float* grad_state, void* workspace, int64_t workspace_bytes, void* stream) {
  return tsfast_hip_gated_bwd_train(B, L, H, Hk, K, V, dtype, q, k, v, g, grad_o, strides, state, grad_last, grad_q, grad_k, grad_v, grad_g, grad_state,
                                    nullptr, workspace, workspace_bytes, stream);
}

int tsfast_hip_gated_step(int64_t B, int64_t H, int64_t Hk, int64_t K, int64_t V, int dtype, const void* q, const void* k, const void* v, const void* g,
                          const int64_t* strides, float* state, void* o, void* stream) {
  if (B < 0 || H < 1 || Hk < 1 || K < 1 || V < 1 || H % Hk != 0 || (dtype != TSF_DTYPE_F32 && dtype != TSF_DTYPE_BF16)) return TSF_ERR_ARG;
  if (K > kStepMaxK || V > (1 << 20) || H > (1 << 20)) return TSF_ERR_UNSUPPORTED;
  if (B == 0) return TSF_OK;
  if (!q || !k || !v || !g || !strides || !state || !o) return TSF_ERR_ARG;
  StepArgs a{q, k, v, g, strides[0], strides[1], strides[2], strides[3], strides[4], strides[5], strides[6], strides[7], state, o,
             (int)H, (int)(H / Hk), (int)K, (int)V, 0};
  const int64_t heads = B * H;
  a.ntile = (int)((V + 4 * kStepLanes - 1) / (4 * kStepLanes));
  if (heads > kMaxGrid / a.ntile) return TSF_ERR_UNSUPPORTED;
  const unsigned grid = (unsigned)(heads * a.ntile);
  if (dtype == TSF_DTYPE_BF16)
    step_kernel<bf16><<<grid, kThreads, 0, (hipStream_t)stream>>>(a);
  else
    step_kernel<float><<<grid, kThreads, 0, (hipStream_t)stream>>>(a);
  return tsf_launch_status();
}

}  // extern "C"
