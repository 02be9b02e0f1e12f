// Gated feed-forward block (gfx950): two projections, an activation and their product, with its gradients.
//
//   a = x Wg^T + bg,  b = x Wu^T + bu,  y = act(a) b          act: silu, gelu (erf) or sigmoid
//   da = dy b act'(a),  db = dy act(a)
//   dx = da Wg + db Wu,  dWg = da^T x,  dWu = db^T x,  dbg = sum da,  dbu = sum db
//
// One kernel, product_kernel, forms the three matrix products: C[q][p] = sum_k Q[q][k] P[p][k], bf16 operands, fp32 sums.
#include <math.h>

#include <type_traits>

#include "common.h"
#include "tsfast_hip.h"

using namespace tsf;

namespace {

constexpr int kThreads = 256;
constexpr int kK = 64;               // of a stage: a row's part is a whole 128-byte line
constexpr int kSlots = 2;            // stages in LDS
constexpr int kMaxSegs = 12;         // products whose sum is formed: 2 sources x 6 pairs of planes
constexpr int64_t kMaxLd = 1 << 22;  // elements between the rows of an operand: 256 rows stay below 2^31 bytes

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4), may_alias));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2), may_alias));

enum Act { kSilu = 0, kGelu = 1, kSigmoid = 2 };
enum Form { kForward = 0, kInput = 1, kWeight = 2 };  // y; dx; dWg and dWu

TSF_DEV uint32_t pack2(float a, float b) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 v = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(uint32_t, v);
}
TSF_DEV float low(uint32_t p) { return __uint_as_float(p << 16); }
TSF_DEV float high(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

// ------------------------------------------------------------------------------------ activations
// The upper tail of the normal distribution, erfc(s) / 2 with s = |a| / sqrt 2, as exp(-s^2) t P(t), t = 1 / (1 + s / 2): P is fitted to the
// least relative error over s <= 12 (7e-8; beyond, the exp is zero in fp32). The exp's argument reaches 122, where its rounding is 2e-5 of the
// exp: nothing beside bf16's 2^-8, but for float32 (T) what a^2 and its product with log2(e) / 2 are rounded by is carried along, so gelu keeps to
// 1e-6 of itself where it is small.
template <int ACT, typename T>
TSF_DEV void activate(float a, float& f, float& df) {
  if constexpr (ACT == kGelu) {
    const float m = fminf(fabsf(a), 16.0f);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.35355339059327376f, m, 1.0f));
    constexpr double kHalf = 0.72134752044448170;  // log2(e) / 2
    constexpr float kHigh = (float)kHalf, kLow = (float)(kHalf - kHigh);
    const float sq = m * m, x = sq * kHigh;
    float e = fast_exp2(-x);
    if constexpr (sizeof(T) == 4) {
      const float rest = fmaf(fmaf(m, m, -sq), kHigh, fmaf(sq, kLow, fmaf(sq, kHigh, -x)));
      e = fmaf(e, -kLn2 * rest, e);
    }
    const float poly = fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, -0.029682316f, 0.14300884f), -0.24509346f), 0.14074159f), -0.014488542f), 0.101840235f), 0.12142658f), 0.14120482f), 0.14104223f);
    const float tail = t * poly * e;
    const float phi = a < 0.0f ? tail : 1.0f - tail;
    f = a * phi;
    df = fmaf(a * 0.39894228040143268f, e, phi);
  } else {
    const float sig = sigmoid_fast(a);
    f = ACT == kSilu ? a * sig : sig;
    df = ACT == kSilu ? fmaf(a * sig, 1.0f - sig, sig) : sig * (1.0f - sig);
  }
}
template <typename T>
TSF_DEV float activate(int act, float a) {
  float f, df;
  if (act == kSilu)
    activate<kSilu, T>(a, f, df);
  else if (act == kGelu)
    activate<kGelu, T>(a, f, df);
  else
    activate<kSigmoid, T>(a, f, df);
  return f;
}

// ------------------------------------------------------------------------------------- operands
// A matrix operand as planes of bf16 whose sum it is: one for bf16 values, three for fp32 ones (8 bits of the mantissa each, split3). Rows
// are 16-byte aligned and their length is a multiple of 8, zeros where the matrix ends before.
struct PackJob {
  const void* src;
  bf16* dst;
  int64_t ld, rows, items;  // items: of 8 columns
  int cols, cols8;
};
struct PackArgs {
  PackJob job[3];
};

// The parts of a float: its nearest bf16 (bf16's largest where that would be infinite), that of what is left, and of what is left then. An
// infinity or NaN is parts (+-1, 0, itself): times a finite factor's parts, and times such a one's, the six products (kPairs) have it exactly
// once or with its own sign, where (itself, 0, 0) would meet the zeros among the factor's parts.
TSF_DEV float lead(float x) {
  constexpr float kMost = 3.3895314e38f;  // bf16's largest
  const float h = fminf(fmaxf((float)(__bf16)x, -kMost), kMost);
  return __builtin_isfinite(x) ? h : copysignf(1.0f, x);
}
TSF_DEV void split3(float x, float* part) {
  const bool finite = __builtin_isfinite(x);
  part[0] = lead(x);
  const float rest = x - part[0];
  part[1] = finite ? rest : 0.0f;
  part[2] = finite ? rest - (float)(__bf16)rest : x;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) pack_kernel(PackArgs a) {
  const PackJob& j = a.job[blockIdx.y];
  const int per = j.cols8 / 8;
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < j.items; i += (int64_t)gridDim.x * kThreads) {
    const int64_t row = i / per;
    const int c = (int)(i % per) * 8;
    const T* src = (const T*)j.src + row * j.ld + c;
    T v[8];
    if (c + 8 <= j.cols) {
      __builtin_memcpy(v, src, sizeof(v));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = c + e < j.cols ? src[e] : from_f32<T>(0.0f);
    }
    bf16* dst = j.dst + row * j.cols8 + c;
    if constexpr (sizeof(T) == 2) {
      __builtin_memcpy(__builtin_assume_aligned(dst, 16), v, 16);
    } else {
      const int64_t plane = j.rows * j.cols8;
      u32x4 w[3];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float p0[3], p1[3];
        split3(v[2 * k], p0);
        split3(v[2 * k + 1], p1);
#pragma unroll
        for (int n = 0; n < 3; ++n) w[n][k] = pack2(p0[n], p1[n]);
      }
#pragma unroll
      for (int n = 0; n < 3; ++n) *(u32x4*)(dst + n * plane) = w[n];
    }
  }
}

// --------------------------------------------------------------------------------- the products
// C[q][p] = sum over segments and k of Q[q][k] P[p][k]. An operand is read as it lies: rows over k, or (a "turned" panel) rows of k over
// its q or p. P comes in two halves of a tile: gate and up rows (forward), or its columns' halves.
struct ProductArgs {
  const bf16 *q[kMaxSegs], *p0[kMaxSegs], *p1[kMaxSegs];
  int64_t ldq, ldp, kq, kp;  // kq, kp: rows of k that each operand has in a segment, as many stages
  int64_t nq, np;           // extent of C (forward: np of each half)
  int64_t tiles_q, tiles_p, stages, split_stages;
  int act, train;
  const void *bg, *bu;      // forward
  void *y, *y1;             // y, dx; dWg and dWu
  float* part;              // sums of each split [split][nq][np] (forward: [split][nq][2][part_ld]), or null
  int64_t part_ld;
  char *save_hi, *save_lo;  // forward of a training step: a and b, see save_pre
  int64_t save_fb;          // blocks of 16 columns
  int64_t half_rows, valid_rows;  // dW: rows of q a half has, and those of them that exist
};

template <int BQ_, int BP_, int WQ_, int WP_>
struct Tile {
  static constexpr int BQ = BQ_, BP = BP_, HP = BP_ / 2, WQ = WQ_, WP = WP_, kWaves = WQ * WP, TH = 64 * kWaves;
  static constexpr int kPerSimd = BQ * BP >= 256 * 256 ? kWaves / 4 : 2;  // waves
  static constexpr int NQ = BQ / WQ / 16, NH = HP / WP / 16;  // 16-row blocks a wave has of q, and of each half of p
  static constexpr int kQBytes = BQ * kK * 2, kHBytes = HP * kK * 2, kStage = kQBytes + 2 * kHBytes;
  static constexpr int kLoads = kStage / 1024 / kWaves;  // 1 KB loads of a wave a stage
  static constexpr int kLds = kSlots * kStage, kOwn = kLds / kWaves;  // a wave's own part, once the products are done
  static_assert(16 * (NH * 16 * 4 + 16) <= kOwn, "");
  static_assert(kStage % (1024 * kWaves) == 0 && kQBytes % 1024 == 0 && kHBytes % 1024 == 0, "");
};

// One 1 KB piece of a panel of ROWS rows (of q or p) x 64 k, by one wave straight into LDS. As it lies: 8 rows of 128 bytes, the eight
// 16-byte chunks of a row turned so that 16 rows' same chunk fall on different banks. Turned: rows of k.
template <int ROWS, bool TURNED>
struct Panel {
  static constexpr int kChunks = ROWS / 8;  // of a row of k
  static constexpr uint32_t kNone = 0x80000000u;
  TSF_DEV static uint32_t swz(uint32_t r) { return (r >> 1) & 7; }
  TSF_DEV static uint32_t turn(uint32_t kr) { return (((kr & 3) << 1) | (((kr >> 3) & 1) << 3)) & (kChunks - 1); }

  uint32_t off, need;  // the lane's byte offset in a stage, and which of the stage's k it starts at
  // `unit`: which 1 KB; rows: of the panel that exist
  TSF_DEV void set(uint32_t unit, uint32_t lane, int64_t ld, uint32_t rows) {
    if constexpr (!TURNED) {
      const uint32_t r = 8 * unit + (lane >> 3), c = (lane & 7) ^ swz(r & 15);
      off = (uint32_t)(r * ld * 2) + c * 16;
      need = r < rows ? c * 8 : ~0u;
    } else {
      constexpr uint32_t per = 64 / kChunks;  // rows of k in 1 KB
      const uint32_t kr = per * unit + lane / kChunks, c = (lane % kChunks) ^ turn(kr);
      off = (uint32_t)(kr * ld * 2) + c * 16;
      need = c * 8 < rows ? kr : ~0u;
    }
  }
  // at: the panel's first row (as it lies: at k = 0, so: bytes from there to the stage's k; turned: the stage's first row of k);
  // left: of the stage's k that exist. A lane whose values do not exist reads beyond the resource's end: zeros.
  TSF_DEV void load(const bf16* at, uint32_t bytes, uint32_t so, uint32_t left, uint32_t to) const {
    const uint32_t v = need < left ? off : kNone;
    const uint64_t a = (uint64_t)at;
    const auto uniform = [](uint32_t v) __attribute__((always_inline)) { return (int)__builtin_amdgcn_readfirstlane(v); };
    const i32x4 rsrc = {uniform((uint32_t)a), uniform((uint32_t)(a >> 32) & 0xffff), uniform(bytes), kBufWord3};
    // Written out, for the compiler makes every later read of LDS wait for the builtin's loads to arrive (vmcnt(0)): no stage would be on its
    // way while the one before is read and multiplied. Only the waits of stage_barrier cover these loads.
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(uniform(to)), "v"(v), "s"(rsrc), "s"(uniform(so)) : "memory", "m0");
  }
  // the bytes from `at` that the lanes which read may reach
  TSF_DEV static uint32_t reach(uint32_t rows, uint32_t k, int64_t ld) {
    return TURNED ? (uint32_t)((kK - 1) * ld + ROWS) * 2 : rows == 0 ? 0 : (uint32_t)((rows - 1) * ld + k) * 2;
  }
};

// The wave's operand blocks of a panel: 16 rows, 8 of the 32 k of a half stage a lane.
template <int ROWS, bool TURNED>
struct Reader {
  using P = Panel<ROWS, TURNED>;
  uint32_t at[2];   // as it lies: the lane's offset in 16 rows, for each half
  uint32_t t, b, m;  // turned: what the chunk is turned by, and the rest of the lane's offset
  TSF_DEV void set(uint32_t li, uint32_t lg) {
    if constexpr (!TURNED) {
      at[0] = li * 128 + ((lg ^ P::swz(li)) << 4);
      at[1] = li * 128 + (((4 + lg) ^ P::swz(li)) << 4);
    } else {
      const uint32_t r = 8 * lg + (li >> 2);
      t = P::turn(r);
      b = r * (ROWS * 2) + 8 * (li & 1);
      m = (li >> 1) & 1;
    }
  }
  TSF_DEV bf16x8 get(const char* panel, uint32_t block, int half) const {
    bf16x8 v;
    if constexpr (!TURNED) {
      const u32x4 w = *(const u32x4*)(panel + block * 2048 + at[half]);
      __builtin_memcpy(&v, &w, 16);
    } else {
      // the transposing read: lane li of a group of 16 points at 4 columns of row li / 4 and receives its own column of the 4
      // rows. Rows 4 and 32 further on are turned alike.
      const char* p = panel + half * 32 * ROWS * 2 + b + (((2 * block + m) ^ t) << 4);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const auto w = __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4*)(
                                                     __attribute__((address_space(3))) char*)const_cast<char*>(p + h * 4 * ROWS * 2)));
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * h + e] = w[e];
      }
    }
    return v;
  }
};

// Waits for all but the last `n` loads into LDS and for this wave's own reads of it, then for the other waves.
template <int N>
TSF_DEV void stage_barrier() {
  __builtin_amdgcn_sched_barrier(0);  // the products before it are issued before it
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

template <typename T>
TSF_DEV void put4(char* p, f32x4 v) {
  if constexpr (sizeof(T) == 2) {
    *(u32x2*)p = u32x2{pack2(v[0], v[1]), pack2(v[2], v[3])};
  } else {
    *(u32x4*)p = __builtin_bit_cast(u32x4, v);
  }
}

// Between a wave's writes of LDS and its other lanes' reads
TSF_DEV void wave_turned() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A wave's part of a half tile of outputs, from accumulators through LDS of the wave's own to memory in whole rows. `row(q)`: the address of
// row q of the wave's rows, or null; n: columns that exist.
template <typename C, typename T, typename V, typename R>
TSF_DEV void store_rows(char* own, uint32_t lane, int n, V value, R row) {
  constexpr int kCols = C::NH * 16, kRow = kCols * (int)sizeof(T) + 16;
  constexpr int kPer = 16 / (int)sizeof(T), kPieces = kCols / kPer;
  const uint32_t li = lane & 15, lg = lane >> 4;
#pragma unroll
  for (int j = 0; j < C::NQ; ++j) {
#pragma unroll
    for (int i = 0; i < C::NH; ++i) put4<T>(own + li * kRow + (i * 16 + 4 * lg) * sizeof(T), value(i, j));
    wave_turned();
#pragma unroll
    for (int e = 0; e < (16 * kPieces + 63) / 64; ++e) {
      const uint32_t at = lane + 64 * e, q = at / kPieces, c = at % kPieces * kPer;
      if (16 * kPieces % 64 != 0 && q >= 16) break;
      T* to = row(16 * j + (int)q);
      if (!to || (int)c >= n) continue;
      const char* from = own + q * kRow + c * sizeof(T);
      if ((int)c + kPer <= n && ((uintptr_t)(to + c) & 15) == 0) {
        __builtin_nontemporal_store(*(const u32x4*)from, (u32x4*)(to + c));
      } else {
#pragma unroll
        for (int k = 0; k < kPer; ++k)
          if ((int)c + k < n) to[c + k] = ((const T*)from)[k];
      }
    }
    wave_turned();
  }
}

// What a training step's forward leaves for its backward: a and b in blocks of 16 rows x 16 columns as accumulators have them (four columns
// a lane). fp32 as it is, 32 bytes a lane; for bf16 the upper 24 bits of each, in 16 bytes (the upper 16 bits of a's and b's) and 8 (the
// next 8). Rounded to bf16 they would cost the gradients as much again as the rounding of da and db does; what is cut off here is below
// 2^-15 of a value.
template <typename T>
TSF_DEV void save_pre(char* hi, char* lo, uint32_t lane, f32x4 a, f32x4 b) {
  if constexpr (sizeof(T) == 4) {
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, a), (u32x4*)(hi + lane * 32));
    __builtin_nontemporal_store(__builtin_bit_cast(u32x4, b), (u32x4*)(hi + lane * 32 + 16));
  } else {
    const u32x4 x = __builtin_bit_cast(u32x4, a), y = __builtin_bit_cast(u32x4, b);
    auto upper = [](uint32_t v1, uint32_t v0) { return __builtin_amdgcn_perm(v1, v0, 0x07060302); };
    auto next = [](const u32x4& v) { return __builtin_amdgcn_perm(__builtin_amdgcn_perm(v[3], v[2], 0x0c0c0501), __builtin_amdgcn_perm(v[1], v[0], 0x0c0c0501), 0x05040100); };
    __builtin_nontemporal_store(u32x4{upper(x[1], x[0]), upper(x[3], x[2]), upper(y[1], y[0]), upper(y[3], y[2])}, (u32x4*)(hi + lane * 16));
    __builtin_nontemporal_store(u32x2{next(x), next(y)}, (u32x2*)(lo + lane * 8));
  }
}
template <typename T>
TSF_DEV void load_pre(const char* hi, const char* lo, int64_t block, uint32_t lane, f32x4& a, f32x4& b) {
  if constexpr (sizeof(T) == 4) {
    const char* p = hi + (block * 64 + lane) * 32;
    a = __builtin_bit_cast(f32x4, *(const u32x4*)p);
    b = __builtin_bit_cast(f32x4, *(const u32x4*)(p + 16));
  } else {
    const u32x4 h = *(const u32x4*)(hi + (block * 64 + lane) * 16);
    const u32x2 l = *(const u32x2*)(lo + (block * 64 + lane) * 8);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint32_t top = e & 1 ? h[e / 2] & 0xffff0000u : h[e / 2] << 16;
      const float v = __uint_as_float(top | ((l[e / 4] >> (8 * (e & 3))) & 0xffu) << 8);
      if (e < 4)
        a[e] = v;
      else
        b[e - 4] = v;
    }
  }
}

// The weights (and, for their gradients, x) are the matrix instruction's first operand: a lane then has four consecutive columns of one row of C.
// A tile of 256 x 256 asks for 8 bytes from memory or L2 per 1024 operations of a stage; two stages of 64 KB are in LDS, one of them on its
// way, and a wave holds the operands of half a stage in registers while it reads the other half's, so the matrix instructions wait for neither.
// Stages of 64 k, not 32, make every load a whole 128-byte line (the three large products 5.4 -> 4.4 ms). What bounds it: the matrix cores at
// the clock that power leaves them (1.6 to 1.8 GHz here), and between a tile's last product and its last store nothing else runs on a CU.
// Measured, 65536 x 1536 -> 2 x 4096 bf16: y with what a backward needs 1.69 ms (980 TFLOP/s), dx 1.30 ms (1270), dWg and dWu 1.35 ms (1220); a
// library product of the same sizes, without the activation and what is kept, 1.40, 1.11 and 1.21 ms. fp32, 16384 x 1536 -> 2 x 4096: packing and y
// 1.78 ms (231 TFLOP/s), a library product of those sizes alone 2.81 ms.
template <typename T, typename C, int FORM>
__global__ void __launch_bounds__(C::TH, C::kPerSimd) product_kernel(ProductArgs g) {
  constexpr bool TQ = FORM == kWeight, TP = FORM != kForward;  // turned operands
  constexpr int NQ = C::NQ, NH = C::NH;
  __shared__ __attribute__((aligned(1024))) char lds[C::kLds];
  const uint32_t tid = threadIdx.x, lane = tid & 63, li = lane & 15, lg = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(tid >> 6), wq = wave / C::WP, wp = wave % C::WP;

  // Workgroups go to the 8 XCDs in turn: each takes a contiguous range of tiles, in groups of 8 tiles of q that share what they read of p.
  const uint32_t total = gridDim.x;
  uint32_t lin = blockIdx.x;
  {
    const uint32_t full = total / 8, rest = total % 8, x = lin % 8, at = lin / 8;
    lin = x * full + (x < rest ? x : rest) + at;
  }
  const uint32_t tiles = (uint32_t)(g.tiles_q * g.tiles_p), split = lin / tiles;
  lin %= tiles;
  const uint32_t gq = 8, group = lin / (gq * (uint32_t)g.tiles_p), first = group * gq;
  const uint32_t in_group = (uint32_t)g.tiles_q - first < gq ? (uint32_t)g.tiles_q - first : gq;
  const uint32_t within = lin - group * gq * (uint32_t)g.tiles_p;
  const int64_t q0 = (int64_t)(first + within % in_group) * C::BQ;
  const int64_t pt = within / in_group;
  const int64_t p0 = pt * (FORM == kForward ? C::HP : C::BP);                 // of the first half
  const int64_t p1 = FORM == kForward ? p0 : p0 + C::HP;                      // of the second
  const uint32_t rows_q = (uint32_t)(g.nq - q0 < C::BQ ? g.nq - q0 : C::BQ);
  const uint32_t rows_0 = (uint32_t)(g.np - p0 < C::HP ? g.np - p0 : C::HP);
  const uint32_t rows_1 = (uint32_t)(g.np - p1 < C::HP ? (g.np > p1 ? g.np - p1 : 0) : C::HP);

  // loads: this wave's pieces of a stage, q's first, then those of p's halves
  constexpr int kQ = C::kQBytes / 1024, kH = C::kHBytes / 1024, kQw = kQ / C::kWaves, kPw = 2 * kH / C::kWaves;
  static_assert(kQw * C::kWaves == kQ && kPw * C::kWaves == 2 * kH, "");
  Panel<C::BQ, TQ> lq[kQw];
  Panel<C::HP, TP> lp[kPw];
  static_assert(kH % C::kWaves == 0, "the wave's pieces of p: as many of each half, the first's first");
  auto half_of = [](int i) __attribute__((always_inline)) { return i / (kPw / 2); };
#pragma unroll
  for (int i = 0; i < kQw; ++i) lq[i].set(wave + i * C::kWaves, lane, g.ldq, rows_q);
#pragma unroll
  for (int i = 0; i < kPw; ++i) lp[i].set((wave + i * C::kWaves) % kH, lane, g.ldp, half_of(i) ? rows_1 : rows_0);
  const int kq = (int)g.kq, kp = (int)g.kp, per_seg = (kq + kK - 1) / kK;
  const int begin = (int)(split * g.split_stages);
  const int count = (int)(g.stages - begin < g.split_stages ? g.stages - begin : g.split_stages);
  int to_load = count, seg = begin / per_seg, k0 = (begin % per_seg) * kK;
  const bf16 *qb, *pb[2];
  auto enter = [&]() __attribute__((always_inline)) {
    qb = g.q[seg] + (TQ ? q0 + k0 * g.ldq : q0 * g.ldq);
    pb[0] = g.p0[seg] + (TP ? p0 + k0 * g.ldp : p0 * g.ldp);
    pb[1] = g.p1[seg] + (TP ? p1 + k0 * g.ldp : p1 * g.ldp);
  };
  enter();
  const uint32_t reach_q = Panel<C::BQ, TQ>::reach(rows_q, kq, g.ldq);
  const uint32_t reach_0 = Panel<C::HP, TP>::reach(rows_0, kp, g.ldp), reach_1 = Panel<C::HP, TP>::reach(rows_1, kp, g.ldp);
  const uint32_t lds_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  // piece i of the next stage, of kLoads; `advance` goes on to the stage after it
  auto load_piece = [&](int buf, int i) __attribute__((always_inline)) {
    const uint32_t to = lds_at + buf * C::kStage + (i < kQw ? 0 : C::kQBytes) + (wave + (i < kQw ? i : i - kQw) * C::kWaves) * 1024;
    const int left = to_load > 0 ? (i < kQw ? kq : kp) - k0 : 0;
    if (i < kQw) {
      lq[i].load(qb, reach_q, TQ ? 0 : k0 * 2, left > 0 ? left : 0, to);
    } else {
      const int n = i - kQw;
      lp[n].load(pb[half_of(n)], half_of(n) ? reach_1 : reach_0, TP ? 0 : k0 * 2, left > 0 ? left : 0, to);
    }
  };
  auto advance = [&]() __attribute__((always_inline)) {
    --to_load;
    k0 += kK;
    if (k0 >= kq && to_load > 0) {
      k0 = 0, ++seg;
      enter();
    } else {
      if (TQ) qb += kK * g.ldq;
      if (TP) pb[0] += kK * g.ldp, pb[1] += kK * g.ldp;
    }
  };

  Reader<C::BQ, TQ> rq;
  Reader<C::HP, TP> rp;
  rq.set(li, lg);
  rp.set(li, lg);
  struct Blocks {
    bf16x8 q[NQ], p[2 * NH];
  };
  // part j, of NQ, of the blocks of a half stage: one of q and as many of p
  constexpr int kPart = 2 * NH / NQ, kEachLoads = C::kLoads / NQ;
  static_assert(kPart * NQ == 2 * NH && kEachLoads * NQ == C::kLoads, "");
  auto read_part = [&](Blocks& f, int slot, int half, int j) __attribute__((always_inline)) {
    const char* from = lds + slot * C::kStage;
#pragma unroll
    for (int i = j * kPart; i < (j + 1) * kPart; ++i) f.p[i] = rp.get(from + C::kQBytes + (i / NH) * C::kHBytes, wp * NH + i % NH, half);
    f.q[j] = rq.get(from, wq * NQ + j, half);
  };
  f32x4 acc[2 * NH][NQ];
#pragma unroll
  for (int i = 0; i < 2 * NH; ++i)
#pragma unroll
    for (int j = 0; j < NQ; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

  auto load_stage = [&](int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < C::kLoads; ++i) load_piece(slot, i);
  };
  // A half stage: its products, from blocks in registers, while the next half's blocks are read from LDS and, in every second one, the
  // stage after the next is loaded into the slot that this stage has left. A wave issues in order, so reads and loads stand evenly
  // between the products: in front of them they would wait for the other waves' first.
  auto half_stage = [&](const Blocks& now, Blocks& next, int read_slot, int half, auto loads, int load_slot) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      if (loads) {
#pragma unroll
        for (int i = 0; i < kEachLoads; ++i) load_piece(load_slot, j * kEachLoads + i);
      }
      read_part(next, read_slot, half, j);
#pragma unroll
      for (int i = 0; i < 2 * NH; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(now.p[i], now.q[j], acc[i][j], 0, 0, 0);
      constexpr int kReads = (TQ ? 2 : 1) + kPart * (TP ? 2 : 1), kEach = 2 * NH / kReads > 0 ? 2 * NH / kReads : 1;
#pragma unroll
      for (int i = 0; i < kReads; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, kEach, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x008, 2 * NH, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  Blocks f0, f1;
  load_stage(0);
  advance();
  load_stage(1);
  stage_barrier<C::kLoads>();
#pragma unroll
  for (int j = 0; j < NQ; ++j) read_part(f0, 0, 0, j);
  for (int t = 0; t < count; ++t) {
    const int slot = t & 1;
    half_stage(f0, f1, slot, 1, std::false_type(), 0);
    advance();
    stage_barrier<0>();  // this stage's slot has been read, the next one's is loaded
    half_stage(f1, f0, slot ^ 1, 0, std::true_type(), slot);
  }
  stage_barrier<0>();

  char* own = lds + wave * C::kOwn;
  auto left = [&](uint32_t columns) { return (int)columns - (int)(wp * NH * 16); };  // of the wave's columns of a half that exist
  if (FORM == kForward && C::BQ < 256 && g.part) {  // join_kernel goes on
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float* y = g.part + (((int64_t)split * g.nq + q0 + wq * NQ * 16) * 2 + h) * g.part_ld + p0 + wp * NH * 16;
      store_rows<C, float>(own, lane, left(rows_0), [&](int i, int j) { return acc[h * NH + i][j]; },
                           [&](int q) { return (uint32_t)q + wq * NQ * 16 < rows_q ? y + q * 2 * g.part_ld : (float*)nullptr; });
    }
  } else if constexpr (FORM == kForward) {
    const T *bg = (const T*)g.bg, *bu = (const T*)g.bu;
    // the wave's first block of 16 rows and of 16 columns, and where a training step keeps it
    const int64_t rb = q0 / 16 + wq * NQ, cb = p0 / 16 + wp * NH, all_rb = (g.nq + 15) / 16, block0 = rb * g.save_fb + cb;
    char *hi = g.save_hi + block0 * (sizeof(T) == 2 ? 1024 : 2048), *lo = g.save_lo + block0 * 512;
    auto finish = [&](auto act) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < NH; ++i) {
        const int64_t f = p0 + (wp * NH + i) * 16 + 4 * lg;
        f32x4 va = {0.0f, 0.0f, 0.0f, 0.0f}, vb = va;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (bg && f + e < g.np) va[e] = to_f32(bg[f + e]);
          if (bu && f + e < g.np) vb[e] = to_f32(bu[f + e]);
        }
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
          f32x4& a = acc[i][j];
          f32x4& b = acc[NH + i][j];
          a += va;
          b += vb;
          if (g.train && rb + j < all_rb && cb + i < g.save_fb) {
            const int64_t block = j * g.save_fb + i;
            save_pre<T>(hi + block * (sizeof(T) == 2 ? 1024 : 2048), lo + block * 512, lane, a, b);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float v, dv;
            activate<decltype(act)::value, T>(a[e], v, dv);
            a[e] = v * b[e];
          }
          __builtin_amdgcn_sched_barrier(0);  // or values of many blocks are alive at once, and spill
        }
      }
    };
    if (g.act == kSilu)
      finish(std::integral_constant<int, kSilu>());
    else if (g.act == kGelu)
      finish(std::integral_constant<int, kGelu>());
    else
      finish(std::integral_constant<int, kSigmoid>());
    const int64_t c0 = p0 + wp * NH * 16;
    T* y = (T*)g.y + (q0 + wq * NQ * 16) * g.np + c0;
    store_rows<C, T>(own, lane, left(rows_0), [&](int i, int j) { return acc[i][j]; },
                     [&](int q) { return (uint32_t)q + wq * NQ * 16 < rows_q ? y + q * g.np : (T*)nullptr; });
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t c0 = (h ? p1 : p0) + wp * NH * 16, r0 = q0 + wq * NQ * 16;
      const int n = left(h ? rows_1 : rows_0);
      auto value = [&](int i, int j) { return acc[h * NH + i][j]; };
      if (g.part) {
        float* y = g.part + ((int64_t)split * g.nq + r0) * g.np + c0;
        store_rows<C, float>(own, lane, n, value, [&](int q) { return (uint32_t)q + wq * NQ * 16 < rows_q ? y + q * g.np : (float*)nullptr; });
      } else if constexpr (FORM == kInput) {
        T* y = (T*)g.y + r0 * g.np + c0;
        store_rows<C, T>(own, lane, n, value, [&](int q) { return (uint32_t)q + wq * NQ * 16 < rows_q ? y + q * g.np : (T*)nullptr; });
      } else {
        store_rows<C, T>(own, lane, n, value, [&](int q) {
          const int64_t r = r0 + q, in = r < g.half_rows ? r : r - g.half_rows;
          T* y = (T*)(r < g.half_rows ? g.y : g.y1);
          return (uint32_t)q + wq * NQ * 16 < rows_q && in < g.valid_rows ? y + in * g.np + c0 : (T*)nullptr;
        });
      }
    }
  }
}

// ------------------------------------------------------------------------------ da and db of dy
// A workgroup has 64 columns and a run of rows; each wave takes every fourth block of 16 rows. da and db go out as the operand planes of
// both products behind, [plane][rows][2 F8], and their column sums as one partial a workgroup.
struct AdjointArgs {
  const void* dy;
  int64_t ld_dy, rows, F, F8, save_fb, blocks;  // blocks: of 16 rows a workgroup has
  const char *save_hi, *save_lo;
  bf16* d;
  float* part;  // [workgroups along rows][2][F], or null
};

// Accumulators hold four columns a lane; memory wants whole lines. A wave's block of 16 rows x 64 columns goes through LDS of its
// own: `kind` of 16 bytes a lane in memory's order, four columns a lane in the accumulators'.
template <typename T>
struct Turn {
  static constexpr int kRow = 64 * (int)sizeof(T) + 16;  // bytes of a row in LDS
  static constexpr int kPer = 16 / (int)sizeof(T), kPieces = 64 / kPer, kEach = 16 * kPieces / 64;
  alignas(16) char at[16 * kRow];
  TSF_DEV static int row(int lane, int e) { return (lane + 64 * e) / kPieces; }
  TSF_DEV static int col(int lane, int e) { return (lane + 64 * e) % kPieces * kPer; }
  TSF_DEV void put_piece(int lane, int e, u32x4 v) { *(u32x4*)(at + row(lane, e) * kRow + col(lane, e) * sizeof(T)) = v; }
  TSF_DEV u32x4 get_piece(int lane, int e) const { return *(const u32x4*)(at + row(lane, e) * kRow + col(lane, e) * sizeof(T)); }
  TSF_DEV void put_four(int li, int c, f32x4 v) { put4<T>(at + li * kRow + c * sizeof(T), v); }
  TSF_DEV f32x4 get_four(int li, int c) const {
    T v[4];
    if constexpr (sizeof(T) == 2) {
      const u32x2 w = *(const u32x2*)(at + li * kRow + c * 2);
      return f32x4{low(w[0]), high(w[0]), low(w[1]), high(w[1])};
    } else {
      return __builtin_bit_cast(f32x4, *(const u32x4*)(at + li * kRow + c * 4));
    }
  }
};

// da = dy b act'(a), db = dy act(a) as planes of bf16 for the two products behind it, rounded once each, and their sums over rows for the
// biases, of the values before that rounding. Bound by memory: 65536 x 4096 bf16 reads 2.1 GB and writes 1.1 GB in 0.67 ms (4.8 TB/s),
// 32768 x 256 fp32 40 us (5.0 TB/s, in part from the cache).
template <typename T, int ACT>
__global__ void __launch_bounds__(kThreads) adjoint_kernel(AdjointArgs g) {
  constexpr int kPlanes = sizeof(T) == 2 ? 1 : 3;
  union Lds {
    Turn<T> dy;
    Turn<bf16> d[2];
  };
  __shared__ Lds lds[4];
  const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, lg = lane >> 4, wave = tid >> 6;
  Lds& turn = lds[wave];
  const int64_t f0 = (int64_t)blockIdx.x * 64, first = (int64_t)blockIdx.y * g.blocks;
  const int64_t all = (g.rows + 15) / 16, last = first + g.blocks < all ? first + g.blocks : all;
  const int64_t plane = g.rows * 2 * g.F8;
  constexpr int kDy = Turn<T>::kEach, kPer = Turn<T>::kPer;
  const int blocks = (int)(g.save_fb - f0 / 16 < 4 ? g.save_fb - f0 / 16 : 4);
  f32x4 sa[4], sb[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) sa[i] = sb[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int64_t mb = first + wave; mb < last; mb += 4) {
    const int64_t m0 = mb * 16;
    f32x4 a[4], b[4];
    u32x4 in[kDy];
    // a load under a lane's condition is waited for before the next one starts: whole blocks have none
    const bool whole = m0 + 16 <= g.rows && f0 + 64 <= g.F;
    const T* dy0 = (const T*)g.dy + m0 * g.ld_dy + f0;
#pragma unroll
    for (int i = 0; i < 4; ++i) load_pre<T>(g.save_hi, g.save_lo, mb * g.save_fb + f0 / 16 + (i < blocks ? i : 0), lane, a[i], b[i]);
    if (whole) {
#pragma unroll
      for (int e = 0; e < kDy; ++e) __builtin_memcpy(&in[e], dy0 + Turn<T>::row(lane, e) * g.ld_dy + Turn<T>::col(lane, e), 16);
    } else {
      const int rows = (int)(g.rows - m0 < 16 ? g.rows - m0 : 16), cols = (int)(g.F - f0 < 64 ? g.F - f0 : 64);
#pragma unroll
      for (int e = 0; e < kDy; ++e) {
        const int r = Turn<T>::row(lane, e), c = Turn<T>::col(lane, e);
        T v[kPer];
#pragma unroll
        for (int k = 0; k < kPer; ++k) v[k] = dy0[(r < rows ? r : rows - 1) * g.ld_dy + (c + k < cols ? c + k : cols - 1)];
#pragma unroll
        for (int k = 0; k < kPer; ++k) v[k] = r < rows && c + k < cols ? v[k] : from_f32<T>(0.0f);
        __builtin_memcpy(&in[e], v, 16);
      }
      // what stands in the place of rows and columns that do not exist may be NaN, which dy = 0 leaves
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool exists = li < rows && 16 * i + 4 * lg + e < cols;
          a[i][e] = exists ? a[i][e] : 0.0f;
          b[i][e] = exists ? b[i][e] : 0.0f;
        }
    }
#pragma unroll
    for (int e = 0; e < kDy; ++e) turn.dy.put_piece(lane, e, in[e]);
    wave_turned();
    f32x4 dy[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) dy[i] = turn.dy.get_four(li, 16 * i + 4 * lg);
    wave_turned();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float v, dv;
        activate<ACT, T>(a[i][e], v, dv);
        a[i][e] = dy[i][e] * dv * b[i][e];  // |dv| < 1.2: no infinity in between that a closed gate (dv = 0) makes NaN
        b[i][e] = dy[i][e] * v;
      }
      sa[i] += a[i];
      sb[i] += b[i];
    }
    // a and b are what is left of da and db from here on; each part of theirs in turn (split3's)
    auto part = [](const f32x4& v, int n) __attribute__((always_inline)) {
      f32x4 p = v;
#pragma unroll
      for (int e = 0; e < 4; ++e) p[e] = kPlanes == 1 || n == 2 ? v[e] : n == 0 ? lead(v[e]) : __builtin_isfinite(v[e]) ? v[e] : 0.0f;
      return p;
    };
#pragma unroll
    for (int n = 0; n < kPlanes; ++n) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 pa = part(a[i], n), pb = part(b[i], n);
        turn.d[0].put_four(li, 16 * i + 4 * lg, pa);
        turn.d[1].put_four(li, 16 * i + 4 * lg, pb);
        if (n + 1 < kPlanes) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            a[i][e] = __builtin_isfinite(a[i][e]) ? a[i][e] - (float)(__bf16)pa[e] : a[i][e];
            b[i][e] = __builtin_isfinite(b[i][e]) ? b[i][e] - (float)(__bf16)pb[e] : b[i][e];
          }
        }
      }
      wave_turned();
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int64_t m = m0 + Turn<bf16>::row(lane, e), f = f0 + Turn<bf16>::col(lane, e);
        if (whole || (m < g.rows && f < g.F8)) {
          bf16* to = g.d + n * plane + m * 2 * g.F8 + f;
          *(u32x4*)to = turn.d[0].get_piece(lane, e);
          *(u32x4*)(to + g.F8) = turn.d[1].get_piece(lane, e);
        }
      }
      wave_turned();
    }
  }
  if (!g.part) return;
  __shared__ float sums[4][2][64];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float x = sa[i][e], y = sb[i][e];
#pragma unroll
      for (int mask = 1; mask < 16; mask <<= 1) x += __shfl_xor(x, mask, kWave), y += __shfl_xor(y, mask, kWave);
      if (li == 0) sums[wave][0][16 * i + 4 * lg + e] = x, sums[wave][1][16 * i + 4 * lg + e] = y;
    }
  __syncthreads();
  if (tid < 128) {
    const int h = tid >> 6, c = tid & 63;
    if (f0 + c < g.F) g.part[((int64_t)blockIdx.y * 2 + h) * g.F + f0 + c] = (sums[0][h][c] + sums[1][h][c]) + (sums[2][h][c] + sums[3][h][c]);
  }
}

// A forward in parts of k: their sums, and what product_kernel does with them otherwise. A wave has a block of 16 rows x 16 columns, four columns a
// lane as accumulators have them.
struct JoinArgs {
  const float* part;  // [splits][rows][2][F8]
  const void *bg, *bu;
  void* y;
  char *save_hi, *save_lo;  // or null
  int64_t rows, F, F8, save_fb;
  int splits, act;
};
template <typename T>
__global__ void __launch_bounds__(kThreads) join_kernel(JoinArgs g) {
  const int lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  const int64_t block = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), rb = block / g.save_fb, cb = block % g.save_fb;
  if (rb * 16 >= g.rows) return;
  const int64_t m = rb * 16 + li, f = cb * 16 + 4 * lg;
  const bool in = m < g.rows && f < g.F;
  const float* p = g.part + (in ? m * 2 * g.F8 + f : 0);
  f32x4 a = {0.0f, 0.0f, 0.0f, 0.0f}, b = a;
#pragma unroll 4
  for (int k = 0; k < g.splits; ++k) {
    a += *(const f32x4*)(p + (int64_t)k * g.rows * 2 * g.F8);
    b += *(const f32x4*)(p + (int64_t)k * g.rows * 2 * g.F8 + g.F8);
  }
  T y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const bool has = in && f + e < g.F;
    a[e] = has ? a[e] + (g.bg ? to_f32(((const T*)g.bg)[f + e]) : 0.0f) : 0.0f;
    b[e] = has ? b[e] + (g.bu ? to_f32(((const T*)g.bu)[f + e]) : 0.0f) : 0.0f;
    y[e] = from_f32<T>(activate<T>(g.act, a[e]) * b[e]);
  }
  if (g.save_hi) save_pre<T>(g.save_hi + block * (sizeof(T) == 2 ? 1024 : 2048), g.save_lo + block * 512, lane, a, b);
  if (!in) return;
  T* to = (T*)g.y + m * g.F + f;
  if (f + 4 <= g.F) {
    __builtin_memcpy(to, y, sizeof(y));
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (f + e < g.F) to[e] = y[e];
  }
}

// What a backward leaves in parts, summed in a fixed order, up to three results in one launch (blockIdx.y): out0 and out1 (or none) [n each] =
// sums over `parts` of part [part][halves][stride] (the first n of each half). VL columns a lane, every fourth part a wave. VL > 1: n and
// stride are multiples of it.
struct SumJob {
  const float* part;
  int64_t stride, n;
  void *out0, *out1;
  int parts, halves;
};
struct SumArgs {
  SumJob job[3];
  int jobs;
  void add(const float* part, int64_t parts, int64_t stride, int64_t n, int halves, void* out0, void* out1) {
    job[jobs++] = SumJob{part, stride, n, out0, out1, (int)parts, halves};
  }
};
template <typename T, int VL>
__global__ void __launch_bounds__(kThreads) sum_kernel(SumArgs a) {
  __shared__ float sums[4][64][VL];
  const SumJob& j = a.job[blockIdx.y];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t i = ((int64_t)blockIdx.x * 64 + lane) * VL, h = i >= j.n, c = i - h * j.n;
  float s[VL];
#pragma unroll
  for (int e = 0; e < VL; ++e) s[e] = 0.0f;
  if (i < j.halves * j.n) {
    const float* p = j.part + h * j.stride + c;
#pragma unroll 4
    for (int k = wave; k < j.parts; k += 4) {
      float v[VL];
      __builtin_memcpy(v, __builtin_assume_aligned(p + (int64_t)k * j.halves * j.stride, 4 * VL), sizeof(v));
#pragma unroll
      for (int e = 0; e < VL; ++e) s[e] += v[e];
    }
  }
#pragma unroll
  for (int e = 0; e < VL; ++e) sums[wave][lane][e] = s[e];
  __syncthreads();
  T* out = (T*)(h ? j.out1 : j.out0);
  if (wave == 0 && i < j.halves * j.n && out) {
#pragma unroll
    for (int e = 0; e < VL; ++e) out[c + e] = from_f32<T>((sums[0][lane][e] + sums[1][lane][e]) + (sums[2][lane][e] + sums[3][lane][e]));
  }
}
template <typename T>
void sum_parts(const SumArgs& a, hipStream_t st) {
  int vl = 4;
  int64_t most = 0;
  for (int k = 0; k < a.jobs; ++k) {
    const SumJob& j = a.job[k];
    if (j.n % 4 || j.stride % 4) vl = 1;
    if (j.halves * j.n > most) most = j.halves * j.n;
  }
  if (most == 0) return;
  auto* const kernel = vl == 4 ? sum_kernel<T, 4> : sum_kernel<T, 1>;
  kernel<<<dim3((unsigned)((most + 64 * vl - 1) / (64 * vl)), (unsigned)a.jobs), kThreads, 0, st>>>(a);
}

// --------------------------------------------------------------------------------- a few rows
// Up to 16 NT rows: the weights are read once and nothing else matters. A workgroup has 16 columns of y; its four waves share the
// contraction, 32 k in turn, both operands straight from memory at any alignment. One row of 1536 -> 2 x 4096 bf16: 6 us, 4.2 TB/s of weights;
// 2048 -> 2 x 8192 fp32 28.5 us, 4.7 TB/s.
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
TSF_DEV f32x4 mma(const Frag<bf16>& a, const Frag<bf16>& b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.v, b.v, c, 0, 0, 0); }
TSF_DEV f32x4 mma(const Frag<float>& a, const Frag<float>& b, f32x4 c) {
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.lo[e], b.lo[e], c, 0, 0, 0);
#pragma unroll
  for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.hi[e], b.hi[e], c, 0, 0, 0);
  return c;
}
// 8 values of a row, the first n of them, zeros after. WHOLE: 8 or none; then loads are unconditional, from k = 0 where there are none: a load
// under a condition is waited for before the next one starts.
template <bool WHOLE, typename T>
TSF_DEV Frag<T> load8(const T* row, int64_t k, int64_t n) {
  T v[8];
  if constexpr (WHOLE) {
    __builtin_memcpy(v, row + (n > 0 ? k : 0), sizeof(v));
    uint32_t w[sizeof(v) / 4];
    __builtin_memcpy(w, v, sizeof(v));
#pragma unroll
    for (int e = 0; e < (int)(sizeof(v) / 4); ++e) w[e] = n > 0 ? w[e] : 0;
    __builtin_memcpy(v, w, sizeof(v));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? row[k + e] : from_f32<T>(0.0f);
  }
  Frag<T> f;
  __builtin_memcpy(&f, v, sizeof(v));
  return f;
}

struct FewArgs {
  const void *x, *wg, *wu, *bg, *bu;
  void* y;
  int64_t rows, D, F, ldx, ldg, ldu;
  int act;
};

template <typename T, int NT, bool WHOLE>
__global__ void __launch_bounds__(kThreads) few_kernel(FewArgs g) {
  __shared__ f32x4 sums[4][2 * NT][64];
  const uint32_t tid = threadIdx.x, lane = tid & 63, li = lane & 15, lg = lane >> 4, wave = tid >> 6;
  const int64_t f0 = (int64_t)blockIdx.x * 16;
  // rows and columns that do not exist repeat the last one: their sums are not used
  const int64_t f = f0 + li < g.F ? f0 + li : g.F - 1;
  const T *wg = (const T*)g.wg + f * g.ldg, *wu = (const T*)g.wu + f * g.ldu;
  const T* x[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) x[t] = (const T*)g.x + (16 * t + li < g.rows ? 16 * t + li : g.rows - 1) * g.ldx;
  f32x4 acc[2][NT];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[h][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int64_t k0 = 32 * wave; k0 < g.D; k0 += 128) {
    const int64_t k = k0 + 8 * lg, n = g.D - k;
    const Frag<T> a = load8<WHOLE>(wg, k, n), b = load8<WHOLE>(wu, k, n);
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const Frag<T> v = load8<WHOLE>(x[t], k, n);
      acc[0][t] = mma(a, v, acc[0][t]);
      acc[1][t] = mma(b, v, acc[1][t]);
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int t = 0; t < NT; ++t) sums[wave][h * NT + t][lane] = acc[h][t];
  __syncthreads();
  // a thread has column tid % 16 of row tid / 16 of each tile of rows: element (column 4 l + e, row li) of lane 16 l + li
  const uint32_t c = tid & 15, r = tid >> 4;
  const int64_t column = f0 + c;
  if (column >= g.F) return;
  const float ba = g.bg ? to_f32(((const T*)g.bg)[column]) : 0.0f, bb = g.bu ? to_f32(((const T*)g.bu)[column]) : 0.0f;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t row = 16 * t + r;
    if (row >= g.rows) continue;
    float v[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t at = (c >> 2) * 16 + r, e = c & 3;
      v[h] = (sums[0][h * NT + t][at][e] + sums[1][h * NT + t][at][e]) + (sums[2][h * NT + t][at][e] + sums[3][h * NT + t][at][e]);
    }
    ((T*)g.y)[row * g.F + column] = from_f32<T>(activate<T>(g.act, v[0] + ba) * (v[1] + bb));
  }
}

// ----------------------------------------------------------------------------------------- host
int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }
int64_t up8(int64_t a) { return up(a, 8) * 8; }
int64_t up256(int64_t a) { return up(a, 256) * 256; }

constexpr int64_t kMaxThreads = ((int64_t)1 << 32) - 1;  // of a launch
// workgroups for n items, one a thread, or as many as a launch has: the kernel strides
int64_t strided(int64_t n) { return up(n, kThreads) < kMaxThreads / kThreads ? up(n, kThreads) : kMaxThreads / kThreads; }

// Rows that few_kernel takes. 33 rows of 2048 -> 2 x 5461 fp32 81 us by product_kernel (45 of them for the planes of the weights), 56 this way
int64_t few_rows(int dtype) { return dtype == TSF_DTYPE_BF16 ? 32 : 64; }

using Large = Tile<256, 256, 4, 2>;
using Medium = Tile<128, 128, 2, 2>;
using Small = Tile<64, 64, 2, 2>;

// How a product of nq x np outputs (forward: np of each half) and `stages` of k is cut: the tile, and the parts of k that side by side
// workgroups take, whichever comes out least. A stage of one workgroup takes `alone` us while its CU has no other, and `shared` us of
// the CU beside others; `ends` is what stands around the stages; the last workgroups' stores, `out_bytes` of each output, have nothing to go on beside.
// Measured, us of the kernel with the large, the medium, the small tile: 256 x 1536 -> 2 x 4096 bf16 36, 20, 16; 1024 rows 39, 29, 43; 2048
// rows 44, 55, 82; 16384 rows with gradients 1200, 1392, 2480. With both operands turned the small tile's stage alone takes longer (dWg
// and dWu of 8192 rows, 256 -> 2 x 1024 bf16, by this rule in medium tiles 19 us, in small ones 23). Partial sums are written and read at
// 4 TB/s. dx of 1000 rows, 768 -> 2 x 2048, whole 33 us, in parts 15 and their sum 2.
struct Plan {
  int tile;  // 0: Large, 1: Medium, 2: Small
  int64_t tiles_q, tiles_p, splits, split_stages;
};
Plan plan_for(Form form, int64_t nq, int64_t np, int64_t stages, int out_bytes) {
  const bool dual = form == kForward;
  const int64_t cus = device_cus();
  const struct {
    int bq, bp, threads, per_cu;
    double alone, shared, ends;
  } tiles[3] = {{Large::BQ, Large::BP, Large::TH, 1, 1.68, 1.68, 8.0},
                {Medium::BQ, Medium::BP, Medium::TH, 2, 0.8, 0.55, 4.0},
                {Small::BQ, Small::BP, Small::TH, 4, form == kWeight ? 0.65 : 0.38, 0.21, 3.0}};
  constexpr double kStore = 18500.0;  // bytes a us of a CU where all store
  Plan best = {};
  double least = 0;
  for (int t = 0; t < 3; ++t) {
    const auto& c = tiles[t];
    const int64_t tq = up(nq, c.bq), tp = up(np, dual ? c.bp / 2 : c.bp);
    for (int64_t s = 1; s <= 64; s *= 2) {
      if (s > 1 && (stages / s < 4 || (dual && t == 0))) break;  // the large tile has no registers to spare for it
      if (tq * tp * s * c.threads > kMaxThreads) break;
      const int64_t wgs = tq * tp * s, round = cus * c.per_cu, full = wgs / round, last = up(wgs % round, cus);
      auto stage = [&](int64_t beside) { return c.alone > beside * c.shared ? c.alone : beside * c.shared; };
      const double each = (double)up(stages, s);
      double time = full * (each * stage(c.per_cu) + c.ends) + (last ? each * stage(last) + c.ends : 0.0);
      if (s == 1) time += (double)(c.bq * c.bp / (dual ? 2 : 1) * out_bytes) / kStore;
      if (s > 1) time += (double)(nq * np * (dual ? 2 : 1) * (2 * s + 1) * 4) / 4e6 + 4.0;
      if (!best.splits || time < least) {
        least = time;
        best = Plan{t, tq, tp, s, up(stages, s)};
      }
    }
  }
  best.splits = up(stages, best.split_stages);
  return best;
}

template <typename T, typename C, int FORM>
void launch_product(ProductArgs& g, const Plan& p, hipStream_t st) {
  product_kernel<T, C, FORM><<<(unsigned)(p.tiles_q * p.tiles_p * p.splits), C::TH, 0, st>>>(g);
}
template <typename T, int FORM>
void product(ProductArgs& g, const Plan& p, hipStream_t st) {
  g.tiles_q = p.tiles_q, g.tiles_p = p.tiles_p, g.split_stages = p.split_stages;
  if (p.tile == 0)
    launch_product<T, Large, FORM>(g, p, st);
  else if (p.tile == 1)
    launch_product<T, Medium, FORM>(g, p, st);
  else
    launch_product<T, Small, FORM>(g, p, st);
}

// An operand's planes: as the matrix lies where its rows are aligned bf16, or packed into the workspace
struct Operand {
  const bf16* p;
  int64_t ld, plane;
  int64_t bytes;  // of the workspace
};
bool lies_well(int dtype, const void* p, int64_t cols, int64_t ld) {
  return dtype == TSF_DTYPE_BF16 && cols % 8 == 0 && ld % 8 == 0 && ((uintptr_t)p & 15) == 0;
}
Operand operand(int dtype, const void* p, int64_t rows, int64_t cols, int64_t ld, bool as_it_lies) {
  if (as_it_lies) return Operand{(const bf16*)p, ld, 0, 0};
  const int64_t planes = dtype == TSF_DTYPE_BF16 ? 1 : 3, c8 = up8(cols);
  return Operand{nullptr, c8, rows * c8, up256(planes * rows * c8 * 2)};
}

// pairs of planes whose products make up that of fp32 matrices to 2^-24, the least first
constexpr int kPairs[6][2] = {{2, 0}, {0, 2}, {1, 1}, {1, 0}, {0, 1}, {0, 0}};

int feed_status(int64_t rows, int64_t D, int64_t F, int dtype, int act) {
  if (rows < 0 || D < 1 || F < 1 || act < 0 || act > 2) return TSF_ERR_ARG;
  if (dtype != TSF_DTYPE_F32 && dtype != TSF_DTYPE_BF16) return TSF_ERR_ARG;
  if (D > kMaxLd / 4 || F > kMaxLd / 4 || rows > ((int64_t)1 << 31) - 64) return TSF_ERR_UNSUPPORTED;
  // every product in one launch: y and dx in the smallest tile, dWg and dWu in the largest (plan_for takes no cut that would be more)
  if (up(rows, Small::BQ) * up(F, Small::HP) > kMaxThreads / Small::TH || up(rows, Small::BQ) * up(D, Small::BP) > kMaxThreads / Small::TH)
    return TSF_ERR_UNSUPPORTED;
  if (up(2 * up8(F), Large::BQ) * up(D, Large::BP) > kMaxThreads / Large::TH) return TSF_ERR_UNSUPPORTED;
  return TSF_OK;
}
bool bad_ld(int64_t ld, int64_t cols) { return ld < cols || ld > kMaxLd; }

int64_t pre_bytes(int64_t rows, int64_t F, int dtype) { return up(rows, 16) * up(F, 16) * 64 * (dtype == TSF_DTYPE_BF16 ? 24 : 32); }
char* pre_lo(char* pre, int64_t rows, int64_t F) { return pre + up(rows, 16) * up(F, 16) * 64 * 16; }

struct Shape {
  int64_t rows, D, F;
  int dtype;
  int64_t F8, stages_f, stages_x, stages_w;  // of the three products
  int pairs;
};
Shape shape_of(int64_t rows, int64_t D, int64_t F, int dtype) {
  Shape s = {rows, D, F, dtype, up8(F), 0, 0, 0, dtype == TSF_DTYPE_BF16 ? 1 : 6};
  s.stages_f = s.pairs * up(D, kK);
  s.stages_x = 2 * s.pairs * up(F, kK);
  s.stages_w = s.pairs * up(rows, kK);
  return s;
}

struct Call {
  const void *x, *wg, *wu;
  int64_t ldx, ldg, ldu;
};
// x and the weights as operands of the products; both weights' rows are equally far apart
struct Operands {
  Operand x, wg, wu;
  int64_t bytes;
};
Operands operands_of(const Shape& s, const Call& c) {
  const bool w = lies_well(s.dtype, c.wg, s.D, c.ldg) && lies_well(s.dtype, c.wu, s.D, c.ldu) && c.ldg == c.ldu;
  Operands o;
  o.x = operand(s.dtype, c.x, s.rows, s.D, c.ldx, lies_well(s.dtype, c.x, s.D, c.ldx));
  o.wg = operand(s.dtype, c.wg, s.F, s.D, c.ldg, w);
  o.wu = operand(s.dtype, c.wu, s.F, s.D, c.ldu, w);
  o.bytes = o.x.bytes + o.wg.bytes + o.wu.bytes;
  return o;
}
// packs what has to be, into ws
template <typename T>
void pack_operands(const Shape& s, const Call& c, Operands& o, char* ws, hipStream_t st) {
  PackArgs a = {};
  int jobs = 0;
  int64_t most = 0;
  auto add = [&](Operand& op, const void* src, int64_t rows, int64_t ld) {
    if (op.p || rows == 0) return;
    op.p = (const bf16*)ws;
    const int64_t items = rows * (op.ld / 8);
    a.job[jobs++] = PackJob{src, (bf16*)ws, ld, rows, items, (int)s.D, (int)op.ld};
    most = items > most ? items : most;
    ws += op.bytes;
  };
  add(o.x, c.x, s.rows, c.ldx);
  add(o.wg, c.wg, s.F, c.ldg);
  add(o.wu, c.wu, s.F, c.ldu);
  if (jobs) pack_kernel<T><<<dim3((unsigned)strided(most), (unsigned)jobs), kThreads, 0, st>>>(a);
}

Plan forward_plan(const Shape& s, bool train) {
  const bool half = s.dtype == TSF_DTYPE_BF16;
  return plan_for(kForward, s.rows, s.F, s.stages_f, (half ? 2 : 4) + (train ? half ? 6 : 8 : 0));
}
int64_t forward_part(const Shape& s, const Plan& p) { return p.splits > 1 ? up256(p.splits * s.rows * 2 * s.F8 * 4) : 0; }

template <typename T, int NT>
void launch_few(const FewArgs& a, hipStream_t st) {
  auto* const kernel = a.D % 8 == 0 ? few_kernel<T, NT, true> : few_kernel<T, NT, false>;
  kernel<<<(unsigned)up(a.F, 16), kThreads, 0, st>>>(a);
}

template <typename T>
int feed_fwd(const Shape& s, const Call& c, int act, const void* bg, const void* bu, void* y, char* pre, char* ws, int64_t ws_bytes, hipStream_t st) {
  if (s.rows <= few_rows(s.dtype) && !pre) {
    const FewArgs a = {c.x, c.wg, c.wu, bg, bu, y, s.rows, s.D, s.F, c.ldx, c.ldg, c.ldu, act};
    if (s.rows <= 16)
      launch_few<T, 1>(a, st);
    else if (s.rows <= 32)
      launch_few<T, 2>(a, st);
    else if constexpr (sizeof(T) == 4)
      launch_few<T, 4>(a, st);
    return tsf_launch_status();
  }
  Operands o = operands_of(s, c);
  const Plan plan = forward_plan(s, pre != nullptr);
  const int64_t bytes = o.bytes + forward_part(s, plan);
  if (bytes && (!ws || ws_bytes < bytes)) return TSF_ERR_WORKSPACE;
  pack_operands<T>(s, c, o, ws, st);
  ProductArgs g = {};
  for (int i = 0; i < s.pairs; ++i) {
    const int* pr = kPairs[s.pairs == 1 ? 5 : i];
    g.q[i] = o.x.p + pr[0] * o.x.plane;
    g.p0[i] = o.wg.p + pr[1] * o.wg.plane;
    g.p1[i] = o.wu.p + pr[1] * o.wu.plane;
  }
  g.ldq = o.x.ld, g.ldp = o.wg.ld, g.kq = g.kp = up8(s.D), g.nq = s.rows, g.np = s.F;
  g.stages = s.stages_f, g.act = act, g.train = pre != nullptr, g.bg = bg, g.bu = bu, g.y = y;
  if (pre) g.save_hi = pre, g.save_lo = pre_lo(pre, s.rows, s.F), g.save_fb = up(s.F, 16);
  if (plan.splits > 1) g.part = (float*)(ws + o.bytes), g.part_ld = s.F8;
  product<T, kForward>(g, plan, st);
  if (g.part) {
    const int64_t fb = up(s.F, 16);
    const JoinArgs j = {g.part, bg, bu, y, g.save_hi, g.save_lo, s.rows, s.F, s.F8, fb, (int)plan.splits, act};
    join_kernel<T><<<(unsigned)up(up(s.rows, 16) * fb, 4), kThreads, 0, st>>>(j);
  }
  return tsf_launch_status();
}

// the parts of a backward's workspace behind the operands
struct BwdSpace {
  Plan px, pw;
  int64_t wgs, blocks;  // of the adjoint's rows
  int64_t d, bias, part_x, part;  // part: of both products, dx's first
};
BwdSpace bwd_space(const Shape& s) {
  BwdSpace b;
  const int size = s.dtype == TSF_DTYPE_BF16 ? 2 : 4;
  b.px = plan_for(kInput, s.rows, s.D, s.stages_x, size);
  b.pw = plan_for(kWeight, 2 * s.F8, s.D, s.stages_w, size);
  const int64_t all = up(s.rows, 16), cols = up(s.F, 64);
  // rows of a workgroup: a block a wave or more (1000 x 2048 bf16 with four at least 23 us, with one 11), and three workgroups a CU, as
  // registers allow: more leave more sums of columns for the next kernel (32768 x 256 fp32: 2048 of them 41 + 14 us, 768 38 + 7)
  b.blocks = up(all * cols, 3 * (int64_t)device_cus());
  if (b.blocks < 4) b.blocks = 4;
  b.wgs = up(all, b.blocks);
  b.d = up256((s.dtype == TSF_DTYPE_BF16 ? 1 : 3) * s.rows * 2 * s.F8 * 2);
  b.bias = up256(b.wgs * 2 * s.F * 4);
  b.part_x = b.px.splits > 1 ? up256(b.px.splits * s.rows * s.D * 4) : 0;
  b.part = b.part_x + (b.pw.splits > 1 ? up256(b.pw.splits * 2 * s.F8 * s.D * 4) : 0);
  return b;
}

template <typename T>
void launch_adjoint(const AdjointArgs& a, int act, dim3 grid, hipStream_t st) {
  if (act == kSilu)
    adjoint_kernel<T, kSilu><<<grid, kThreads, 0, st>>>(a);
  else if (act == kGelu)
    adjoint_kernel<T, kGelu><<<grid, kThreads, 0, st>>>(a);
  else
    adjoint_kernel<T, kSigmoid><<<grid, kThreads, 0, st>>>(a);
}

template <typename T>
int feed_bwd(const Shape& s, const Call& c, int act, const void* dy, int64_t ld_dy, const char* pre, void* dx, void* dwg, void* dwu, void* dbg,
             void* dbu, char* ws, int64_t ws_bytes, hipStream_t st) {
  Operands o = operands_of(s, c);
  const BwdSpace b = bwd_space(s);
  if (!ws || ws_bytes < o.bytes + b.d + b.bias + b.part) return TSF_ERR_WORKSPACE;
  pack_operands<T>(s, c, o, ws, st);
  char* at = ws + o.bytes;
  bf16* d = (bf16*)at;
  float* bias = (float*)(at + b.d);
  float* part_x = (float*)(at + b.d + b.bias);
  float* part_w = (float*)(at + b.d + b.bias + b.part_x);
  SumArgs sums = {};
  const bool want_bias = dbg || dbu;

  AdjointArgs a = {};
  a.dy = dy, a.ld_dy = ld_dy, a.rows = s.rows, a.F = s.F, a.F8 = s.F8, a.save_fb = up(s.F, 16), a.blocks = b.blocks;
  a.save_hi = pre, a.save_lo = pre_lo(const_cast<char*>(pre), s.rows, s.F), a.d = d, a.part = want_bias ? bias : nullptr;
  launch_adjoint<T>(a, act, dim3((unsigned)up(s.F, 64), (unsigned)b.wgs), st);
  if (want_bias) sums.add(bias, b.wgs, s.F, s.F, 2, dbg, dbu);

  const int64_t plane = s.rows * 2 * s.F8;
  if (dx) {
    ProductArgs g = {};
    for (int src = 0; src < 2; ++src)
      for (int i = 0; i < s.pairs; ++i) {
        const int* pr = kPairs[s.pairs == 1 ? 5 : i];
        const Operand& w = src ? o.wu : o.wg;
        const int n = src * s.pairs + i;
        g.q[n] = d + pr[0] * plane + src * s.F8;
        g.p0[n] = g.p1[n] = w.p + pr[1] * w.plane;
      }
    g.ldq = 2 * s.F8, g.ldp = o.wg.ld, g.kq = s.F8, g.kp = s.F, g.nq = s.rows, g.np = s.D;
    g.stages = s.stages_x, g.y = dx, g.part = b.px.splits > 1 ? part_x : nullptr;
    product<T, kInput>(g, b.px, st);
    if (g.part) sums.add(g.part, b.px.splits, s.rows * s.D, s.rows * s.D, 1, dx, nullptr);
  }
  if (dwg || dwu) {
    ProductArgs g = {};
    for (int i = 0; i < s.pairs; ++i) {
      const int* pr = kPairs[s.pairs == 1 ? 5 : i];
      g.q[i] = d + pr[0] * plane;
      g.p0[i] = g.p1[i] = o.x.p + pr[1] * o.x.plane;
    }
    g.ldq = 2 * s.F8, g.ldp = o.x.ld, g.kq = g.kp = s.rows, g.nq = 2 * s.F8, g.np = s.D;
    g.stages = s.stages_w, g.y = dwg, g.y1 = dwu, g.half_rows = s.F8, g.valid_rows = s.F;
    g.part = b.pw.splits > 1 ? part_w : nullptr;
    product<T, kWeight>(g, b.pw, st);
    if (g.part) sums.add(g.part, b.pw.splits, s.F8 * s.D, s.F * s.D, 2, dwg, dwu);
  }
  sum_parts<T>(sums, st);
  return tsf_launch_status();
}

template <typename T>
__global__ void __launch_bounds__(kThreads) zero_kernel(T* p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) p[i] = from_f32<T>(0.0f);
}
template <typename T>
void zero(void* p, int64_t n, hipStream_t st) {
  if (p && n > 0) zero_kernel<T><<<(unsigned)strided(n), kThreads, 0, st>>>((T*)p, n);
}

}  // namespace

extern "C" {

int tsfast_hip_feed_plan(int64_t rows, int64_t D, int64_t F, int dtype, int train, int64_t* plan) {
  const int rc = feed_status(rows, D, F, dtype, 0);
  if (rc != TSF_OK) return rc;
  if (rows == 0 || !plan) return TSF_ERR_ARG;
  const Shape s = shape_of(rows, D, F, dtype);
  const BwdSpace b = bwd_space(s);
  const int edge[3] = {Large::BQ, Medium::BQ, Small::BQ}, threads[3] = {Large::TH, Medium::TH, Small::TH};
  int64_t* to = plan;
  for (const Plan& p : {forward_plan(s, train), b.px, b.pw}) *to++ = edge[p.tile], *to++ = p.splits, *to++ = p.tiles_q * p.tiles_p * p.splits, *to++ = threads[p.tile];
  if (rows <= few_rows(dtype) && !train) plan[0] = 0, plan[1] = 1, plan[2] = up(F, 16), plan[3] = kThreads;
  return TSF_OK;
}

int64_t tsfast_hip_feed_kept_bytes(int64_t rows, int64_t D, int64_t F, int dtype) {
  if (feed_status(rows, D, F, dtype, 0) != TSF_OK) return -1;
  return pre_bytes(rows, F, dtype);
}

int64_t tsfast_hip_feed_fwd_workspace_bytes(int64_t rows, int64_t D, int64_t F, int dtype, const void* x, int64_t x_stride, const void* w_gate,
                                            int64_t w_gate_stride, const void* w_up, int64_t w_up_stride, int train) {
  if (feed_status(rows, D, F, dtype, 0) != TSF_OK) return -1;
  if (rows <= few_rows(dtype) && !train) return 0;
  if (rows == 0) return 0;
  const Shape s = shape_of(rows, D, F, dtype);
  return operands_of(s, Call{x, w_gate, w_up, x_stride, w_gate_stride, w_up_stride}).bytes + forward_part(s, forward_plan(s, train));
}

int64_t tsfast_hip_feed_bwd_workspace_bytes(int64_t rows, int64_t D, int64_t F, int dtype, const void* x, int64_t x_stride, const void* w_gate,
                                            int64_t w_gate_stride, const void* w_up, int64_t w_up_stride) {
  if (feed_status(rows, D, F, dtype, 0) != TSF_OK) return -1;
  if (rows == 0) return 0;
  const Shape s = shape_of(rows, D, F, dtype);
  const BwdSpace b = bwd_space(s);
  return operands_of(s, Call{x, w_gate, w_up, x_stride, w_gate_stride, w_up_stride}).bytes + b.d + b.bias + b.part;
}

int tsfast_hip_feed_fwd(int64_t rows, int64_t D, int64_t F, int dtype, int activation, const void* x, int64_t x_stride, const void* w_gate,
                        int64_t w_gate_stride, const void* w_up, int64_t w_up_stride, const void* b_gate, const void* b_up, void* y, void* kept,
                        void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = feed_status(rows, D, F, dtype, activation);
  if (rc != TSF_OK) return rc;
  if (rows == 0) return TSF_OK;
  if (!x || !w_gate || !w_up || !y) return TSF_ERR_ARG;
  if (bad_ld(x_stride, D) || bad_ld(w_gate_stride, D) || bad_ld(w_up_stride, D)) return TSF_ERR_ARG;
  const Shape s = shape_of(rows, D, F, dtype);
  const Call c = {x, w_gate, w_up, x_stride, w_gate_stride, w_up_stride};
  auto* f = dtype == TSF_DTYPE_BF16 ? feed_fwd<bf16> : feed_fwd<float>;
  return f(s, c, activation, b_gate, b_up, y, (char*)kept, (char*)workspace, workspace_bytes, (hipStream_t)stream);
}

int tsfast_hip_feed_bwd(int64_t rows, int64_t D, int64_t F, int dtype, int activation, const void* x, int64_t x_stride, const void* w_gate,
                        int64_t w_gate_stride, const void* w_up, int64_t w_up_stride, const void* grad_y, int64_t grad_y_stride,
                        const void* kept, void* grad_x, void* grad_w_gate, void* grad_w_up, void* grad_b_gate, void* grad_b_up, void* workspace,
                        int64_t workspace_bytes, void* stream) {
  const int rc = feed_status(rows, D, F, dtype, activation);
  if (rc != TSF_OK) return rc;
  const hipStream_t st = (hipStream_t)stream;
  if (rows == 0) {
    auto* z = dtype == TSF_DTYPE_BF16 ? zero<bf16> : zero<float>;
    z(grad_w_gate, F * D, st), z(grad_w_up, F * D, st), z(grad_b_gate, F, st), z(grad_b_up, F, st);
    return tsf_launch_status();
  }
  if (!x || !w_gate || !w_up || !grad_y || !kept || !grad_w_gate != !grad_w_up) return TSF_ERR_ARG;
  if (bad_ld(x_stride, D) || bad_ld(w_gate_stride, D) || bad_ld(w_up_stride, D) || grad_y_stride < F) return TSF_ERR_ARG;
  const Shape s = shape_of(rows, D, F, dtype);
  const Call c = {x, w_gate, w_up, x_stride, w_gate_stride, w_up_stride};
  auto* f = dtype == TSF_DTYPE_BF16 ? feed_bwd<bf16> : feed_bwd<float>;
  return f(s, c, activation, grad_y, grad_y_stride, (const char*)kept, grad_x, grad_w_gate, grad_w_up, grad_b_gate, grad_b_up, (char*)workspace,
           workspace_bytes, st);
}

}  // extern "C"
