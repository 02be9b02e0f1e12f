// A Mamba layer's convolution and scan over sequences packed into one row of tokens, in service (gfx950).
//
//   u_t   = silu(bias + sum_k w_k x_{t-(K-1)+k})            left of a sequence's first token: its carried tail
//   h_t   = exp(delta_t A) h_{t-1} + delta_t u_t B_t,       delta = softplus(draw)
//   out_t = (sum_n h_t C_t + Dp u_t) silu(z_t)              h before a sequence's first token: its carried state
//
// Sequence s has the tokens starts[s] .. starts[s + 1) of T; a sequence may be empty. The states that a sequence leaves (its
// last K - 1 inputs; h after its last token) go out for the steps token by token behind it. Tokens without a sequence give zeros.
// starts is read on the device: the host knows T and S only. Whatever starts holds, no access leaves the tensors and every loop ends.
#include "common.h"
#include "tsfast_hip.h"

using namespace tsf;

namespace {

constexpr int kThreads = 256;
constexpr int kMaxK = 8;

// ---------------------------------------------------------------------------------- the sequences
struct Starts {
  const void* p;
  int wide;  // int64, else int32
  int S, T;
  // where sequence s begins (s = S: where the last one ends), within the tokens there are
  TSF_DEV int at(int64_t s) const {
    const int64_t v = wide ? ((const int64_t*)p)[s] : (int64_t)((const int32_t*)p)[s];
    return v < 0 ? 0 : v > T ? T : (int)v;
  }
};

// A token's sequence: the last one that begins at or before it (so it is not empty); -1: none yet, S: behind the last one. Where it begins
// and ends: before and behind the sequences, where no token has one. begin <= t even where starts decreases: what is addressed by
// t - begin, or by the segment before t's, exists.
struct Cursor {
  int s, begin, end;
  // for a token of each lane; all lanes of a wave call. Up to 64 starts come with one load of the wave (a search is a chain of loads)
  TSF_DEV void find(const Starts& st, int t, int lane) {
    if (st.S < 64) {
      const int mine = st.at(lane < st.S ? lane : st.S);
      int count = 0;
      for (int l = 0; l <= st.S; ++l) count += __builtin_amdgcn_readlane(mine, l) <= t;
      s = count - 1;
      const int from = __shfl(mine, s < 0 ? 0 : s, kWave);
      begin = s < 0 ? 0 : from < t ? from : t;
      end = __shfl(mine, s < st.S ? s + 1 : st.S, kWave);
    } else {
      int lo = 0, hi = st.S + 1;  // the first start behind t is in [lo, hi]
      while (lo < hi) {
        const int mid = lo + (hi - lo) / 2;
        if (st.at(mid) <= t)
          lo = mid + 1;
        else
          hi = mid;
      }
      s = lo - 1;
      begin = s < 0 ? 0 : st.at(s);
      end = st.at(s < st.S ? s + 1 : st.S);
    }
    if (s >= st.S) end = st.T;
  }
  // the same token in all lanes: scalar registers
  TSF_DEV void find_uniform(const Starts& st, int t, int lane) {
    find(st, t, lane);
    s = __builtin_amdgcn_readfirstlane(s), begin = __builtin_amdgcn_readfirstlane(begin), end = __builtin_amdgcn_readfirstlane(end);
  }
  TSF_DEV bool has(const Starts& st) const { return s >= 0 && s < st.S; }
  // to the next sequence that is not over at t, or behind the last one; the present one is over
  TSF_DEV void next(const Starts& st, int t) {
    do {
      ++s;
      begin = end;
      end = s < st.S ? st.at(s + 1) : st.T;
    } while (s < st.S && end <= t);
  }
};

// ------------------------------------------------------------------------------------ convolution
// A thread has 16 bytes of channels (8 bf16, 4 fp32) and RUN tokens. Where no sequence begins or ends within or right before them, all of its
// rows are loaded at once; elsewhere it goes token by token. 16384 x 1536 bf16: 30 us with 24 sequences, 26 with one, of 21 that a copy of
// its bytes takes.
struct ConvArgs {
  const void *x, *tails, *weight, *bias;
  void *out, *tails_out;
  int64_t D, sx, groups, runs;  // groups of channels; runs of tokens
  Starts starts;
  int w_bf16, b_bf16;
};
TSF_DEV float param(const void* p, int64_t i, int is_bf16) { return is_bf16 ? to_f32(((const bf16*)p)[i]) : ((const float*)p)[i]; }

template <typename T, int VL>
TSF_DEV void load_row(float* v, const T* p, int n) {
  T h[VL];
  if (n >= VL) {
    __builtin_memcpy(h, p, sizeof(h));
  } else {
#pragma unroll
    for (int e = 0; e < VL; ++e) h[e] = e < n ? p[e] : from_f32<T>(0.0f);
  }
#pragma unroll
  for (int e = 0; e < VL; ++e) v[e] = to_f32(h[e]);
}
template <typename T, int VL>
TSF_DEV void store_row(T* p, const float* v, int n) {
  T h[VL];
#pragma unroll
  for (int e = 0; e < VL; ++e) h[e] = from_f32<T>(v[e]);
  if (n >= VL) {
    __builtin_memcpy(p, h, sizeof(h));
  } else {
#pragma unroll
    for (int e = 0; e < VL; ++e)
      if (e < n) p[e] = h[e];
  }
}

template <typename T, int K, int RUN>
__global__ void __launch_bounds__(kThreads) conv_kernel(ConvArgs g) {
  constexpr int VL = 16 / (int)sizeof(T);
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t run = i / g.groups, c0 = (i % g.groups) * VL;
  const int n = (int)(g.D - c0 < VL ? g.D - c0 : VL), S = g.starts.S, T_all = g.starts.T;
  const T *x = (const T*)g.x + c0, *tails = (const T*)g.tails;
  T *out = (T*)g.out + c0, *tails_out = (T*)g.tails_out;
  const int t0 = run < g.runs ? (int)run * RUN : 0, t1 = t0 + RUN < T_all ? t0 + RUN : T_all;
  Cursor at;
  at.find(g.starts, t0, threadIdx.x & 63);
  if (run >= g.runs) {  // an empty sequence leaves what it was given
    const int64_t s = run - g.runs;
    if (s >= S || g.starts.at(s + 1) > g.starts.at(s)) return;
    const int64_t to = (s * g.D + c0) * (K - 1);
    for (int e = 0; e < n * (K - 1); ++e) tails_out[to + e] = tails ? tails[to + e] : from_f32<T>(0.0f);
    return;
  }
  float w[K][VL], b[VL];
#pragma unroll
  for (int e = 0; e < VL; ++e) {
    const int64_t c = c0 + (e < n ? e : n - 1);
    b[e] = g.bias ? param(g.bias, c, g.b_bf16) : 0.0f;
  }
  if (g.w_bf16) {
#pragma unroll
    for (int e = 0; e < VL; ++e)
#pragma unroll
      for (int k = 0; k < K; ++k) w[k][e] = to_f32(((const bf16*)g.weight)[(c0 + (e < n ? e : n - 1)) * K + k]);
  } else {
#pragma unroll
    for (int e = 0; e < VL; ++e)
#pragma unroll
      for (int k = 0; k < K; ++k) w[k][e] = ((const float*)g.weight)[(c0 + (e < n ? e : n - 1)) * K + k];
  }
  if (at.has(g.starts) && at.begin <= t0 - (K - 1) && at.end > t1 && t1 - t0 == RUN && n == VL) {
    T rows[RUN + K - 1][VL];
#pragma unroll
    for (int k = 0; k < RUN + K - 1; ++k) __builtin_memcpy(rows[k], x + (int64_t)(t0 - (K - 1) + k) * g.sx, sizeof(rows[k]));
#pragma unroll
    for (int k = 0; k < RUN; ++k) {
      float y[VL];
#pragma unroll
      for (int e = 0; e < VL; ++e) {
        float a = b[e];
#pragma unroll
        for (int j = 0; j < K; ++j) a = fmaf(w[j][e], to_f32(rows[k + j][e]), a);
        y[e] = a * sigmoid_fast(a);
      }
      store_row<T, VL>(out + (int64_t)(t0 + k) * g.D, y, VL);
    }
    return;
  }
  float past[K - 1][VL] = {};  // past[k]: the input K - 1 - k tokens ago
  // tail value k of the present sequence
  auto carried = [&](int k, int e) __attribute__((always_inline)) {
    return tails && e < n ? to_f32(tails[((int64_t)at.s * g.D + c0 + e) * (K - 1) + k]) : 0.0f;
  };
  if (at.has(g.starts)) {
#pragma unroll
    for (int k = 0; k < K - 1; ++k) {
      const int t = t0 - (K - 1) + k;
      if (t >= at.begin) {
        load_row<T, VL>(past[k], x + (int64_t)t * g.sx, n);
      } else {
        const int from = t - at.begin + (K - 1);  // in [0, K - 1): t0 >= begin
#pragma unroll
        for (int e = 0; e < VL; ++e) past[k][e] = carried(from, e);
      }
    }
  }
  T rows[RUN][VL];  // all at once: a row that does not exist repeats the last one
  if (n == VL) {
#pragma unroll
    for (int i = 0; i < RUN; ++i) __builtin_memcpy(rows[i], x + (int64_t)(t0 + i < T_all ? t0 + i : T_all - 1) * g.sx, sizeof(rows[i]));
  } else {
#pragma unroll
    for (int i = 0; i < RUN; ++i)
#pragma unroll
      for (int e = 0; e < VL; ++e) rows[i][e] = x[(int64_t)(t0 + i < T_all ? t0 + i : T_all - 1) * g.sx + (e < n ? e : n - 1)];
  }
#pragma unroll
  for (int i = 0; i < RUN; ++i) {
    const int t = t0 + i;
    if (t < t1) {
      if (t >= at.end) {
        at.next(g.starts, t);
        if (at.has(g.starts)) {
#pragma unroll
          for (int k = 0; k < K - 1; ++k)
#pragma unroll
            for (int e = 0; e < VL; ++e) past[k][e] = carried(k, e);
        }
      }
      const bool has = at.has(g.starts);
      float y[VL];
#pragma unroll
      for (int e = 0; e < VL; ++e) {
        float a = b[e];
#pragma unroll
        for (int k = 0; k < K - 1; ++k) a = fmaf(w[k][e], past[k][e], a);
        a = fmaf(w[K - 1][e], to_f32(rows[i][e]), a);
        y[e] = has ? a * sigmoid_fast(a) : 0.0f;
#pragma unroll
        for (int k = 0; k < K - 1; ++k) past[k][e] = k + 1 < K - 1 ? past[k + 1 < K - 1 ? k + 1 : k][e] : to_f32(rows[i][e]);
      }
      store_row<T, VL>(out + (int64_t)t * g.D, y, n);
      if (has && t == at.end - 1) {
#pragma unroll
        for (int e = 0; e < VL; ++e)
#pragma unroll
          for (int k = 0; k < K - 1; ++k)
            if (e < n) tails_out[((int64_t)at.s * g.D + c0 + e) * (K - 1) + k] = from_f32<T>(past[k][e]);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------ scan
// A workgroup has 64 channels and a run of tokens (a segment). Each of its four waves has a quarter of the states of all 64, a
// channel a lane, in registers; what depends on a token and a channel (softplus, gates) is done once, by the thread that owns the pair,
// and goes through LDS, a chunk of kTok tokens at a time. Vector instructions bound it: a token's state is about six
// issue slots (its exp two) and a share of some thirty of a token and channel, 95 us for 16384 x 1536 x 16 at 2.4 GHz, where the walk takes 123;
// segments' maps have to form the same exps before (70, takes 85), and the join is 11. Memory would allow 45 us. A short row is the latency of its tokens, 0.15 us each.
constexpr int kTok = 16;
constexpr int kCh = 64;
struct ScanArgs {
  const void *draw, *Bt, *Ct, *u, *z;
  const float *A, *Dp, *h0;
  void* out;
  float* h_last;
  int64_t sdraw, sb, sc, su, sz;  // distances between tokens
  int64_t D, tiles, seg_len, segs;
  int N;
  Starts starts;
  float* maps;  // of segments: sums of delta [segs][D], then states [segs][N][D]
};

// Waves a SIMD that the registers are to allow where a wave has states that do not exist: what they allow by themselves where it has none.
constexpr int scan_waves(int npt) { return npt >= 16 ? 3 : npt >= 8 ? 4 : npt >= 2 ? 5 : 4; }

// The walk of one segment. ALL: N = 4 NPT, every state exists. MAP: only the state it hands to the next one, from the last sequence's first token in it (or its own
// first token with no state), with the sum of delta that decays what enters; -1: nothing that enters reaches the next segment.
template <typename T, int NPT, bool MAP, bool ALL>
__global__ void __launch_bounds__(kThreads, ALL ? 1 : scan_waves(NPT)) scan_kernel(ScanArgs g) {
  __shared__ float2 s_sc[kTok][kCh];         // delta, delta u
  __shared__ float2 s_bc[kTok][4 * NPT];     // B, C
  __shared__ float s_y[MAP ? 1 : kTok][4][kCh];  // each wave's sum over its states
  __shared__ int s_odd[2];                       // whether a chunk has an infinite or NaN delta u; chunks in turn
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t tile = blockIdx.x % g.tiles, seg = blockIdx.x / g.tiles, d = tile * kCh + lane;
  const int S = g.starts.S, T_all = g.starts.T;
  const int N = g.N, n0 = wave * NPT;
  const bool act = d < g.D;
  int t0 = (int)(seg * g.seg_len);
  const int t1 = t0 + g.seg_len < T_all ? (int)(t0 + g.seg_len) : T_all;

  float A2[NPT], h[NPT];
#pragma unroll
  for (int j = 0; j < NPT; ++j) A2[j] = act && n0 + j < N ? g.A[d * N + n0 + j] * kLog2e : 0.0f, h[j] = 0.0f;
  auto begin_state = [&](int64_t s) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NPT; ++j) h[j] = g.h0 && act && n0 + j < N ? g.h0[(s * g.D + d) * N + n0 + j] : 0.0f;
  };
  auto end_state = [&](int64_t s) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < NPT; ++j)
      if (act && n0 + j < N) g.h_last[(s * g.D + d) * N + n0 + j] = h[j];
  };

  Cursor at;
  bool whole = false;
  if (MAP) {
    // the sequence that goes on in the next segment, if one does
    at.find_uniform(g.starts, t1 - 1, lane);
    if (!at.has(g.starts) || t1 >= T_all || at.end <= t1) return;
    whole = at.begin < t0;  // the segment lies within the sequence
    if (!whole) {
      t0 = at.begin;
      begin_state(at.s);
    }
  } else {
    // sequences without a token leave what they were given
    for (int64_t e = seg; e < S; e += g.segs)
      if (g.starts.at(e + 1) <= g.starts.at(e)) begin_state(e), end_state(e);
    at.find_uniform(g.starts, t0, lane);
#pragma unroll
    for (int j = 0; j < NPT; ++j) h[j] = 0.0f;
    if (at.has(g.starts)) {
      if (at.begin == t0) {
        begin_state(at.s);
      } else {
        const float* from = g.maps + g.segs * g.D + (seg - 1) * N * g.D;
#pragma unroll
        for (int j = 0; j < NPT; ++j) h[j] = act && n0 + j < N ? from[(n0 + j) * g.D + d] : 0.0f;
      }
    }
  }

  constexpr int kOwn = kTok / 4;  // tokens of its channel that a thread owns in a chunk: wave + 4 k
  constexpr int kBc = (kTok * 4 * NPT + kThreads - 1) / kThreads;
  struct Chunk {
    T dr[kOwn], u[kOwn], z[kOwn], b[kBc], c[kBc];
  };
  // two chunks ahead. Tokens, channels and states that do not exist repeat the last one, so that no load stands under a condition
  const int64_t dc = act ? d : g.D - 1;
  auto load = [&](Chunk& r, int tc) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
      const int i = tc + wave + 4 * k;
      const int64_t t = i < t1 ? i : t1 - 1;
      r.dr[k] = ((const T*)g.draw)[t * g.sdraw + dc];
      r.u[k] = ((const T*)g.u)[t * g.su + dc];
      if (!MAP) r.z[k] = ((const T*)g.z)[t * g.sz + dc];
    }
#pragma unroll
    for (int k = 0; k < kBc; ++k) {
      const int i = tid + k * kThreads, n = i % (4 * NPT), m = tc + i / (4 * NPT);
      const int64_t t = m < t1 ? m : t1 - 1;
      const int nc = n < N ? n : N - 1;
      r.b[k] = ((const T*)g.Bt)[t * g.sb + nc];
      if (!MAP) r.c[k] = ((const T*)g.Ct)[t * g.sc + nc];
    }
  };
  const float dp = !MAP && act ? g.Dp[d] : 0.0f;
  const int first = g.starts.at(0), last = g.starts.at(S);  // tokens that have a sequence
  float sum = 0.0f;
  auto chunk = [&](Chunk& r, int tc, int turn) __attribute__((always_inline)) {
    const int len = t1 - tc < kTok ? t1 - tc : kTok;
    bool odd = false;
    float o_u[kOwn], o_z[kOwn];
#pragma unroll
    for (int k = 0; k < kOwn; ++k) {
      const int i = wave + 4 * k;
      o_u[k] = to_f32(r.u[k]);
      if (!MAP) o_z[k] = to_f32(r.z[k]);
      const float delta = i < len ? softplus_fast(to_f32(r.dr[k])) : 0.0f;  // nothing is done with tokens past the end
      if (MAP) sum += delta;
      s_sc[i][lane] = make_float2(delta, delta * o_u[k]);
      odd = odd || !__builtin_isfinite(delta * o_u[k]);
    }
    if (!ALL && odd) s_odd[turn] = 1;
#pragma unroll
    for (int k = 0; k < kBc; ++k) {
      const int i = tid + k * kThreads;
      if (kTok * 4 * NPT % kThreads == 0 || i < kTok * 4 * NPT)
        s_bc[i / (4 * NPT)][i % (4 * NPT)] = i % (4 * NPT) < N ? make_float2(to_f32(r.b[k]), MAP ? 0.0f : to_f32(r.c[k])) : make_float2(0.0f, 0.0f);
    }
    load(r, tc + 2 * kTok);
    __syncthreads();
    auto step = [&](int i) __attribute__((always_inline)) {
      const float2 sc = s_sc[i][lane];
      float y = 0.0f;
#pragma unroll
      for (int j = 0; j < NPT; ++j) {
        const float2 bc = s_bc[i][n0 + j];
        h[j] = fmaf(fast_exp2(sc.x * A2[j]), h[j], sc.y * bc.x);
        y = fmaf(h[j], bc.y, y);
      }
      if (!MAP) s_y[i][wave][lane] = y;
    };
    // Beside an infinite or NaN delta u the zeros of states that do not exist would be NaN among the sums: there, without them. 16384 x 1536 with 17
    // states 304 us, with 40 575 (without this path 302 and 549; with masks in every chunk instead 40 states took 800).
    auto step_without = [&](int i) __attribute__((always_inline)) {
      const float2 sc = s_sc[i][lane];
      float y = 0.0f;
#pragma unroll
      for (int j = 0; j < NPT; ++j) {
        const float2 bc = s_bc[i][n0 + j];
        h[j] = n0 + j < N ? fmaf(fast_exp2(sc.x * A2[j]), h[j], sc.y * bc.x) : 0.0f;
        y = n0 + j < N ? fmaf(h[j], bc.y, y) : y;
      }
      s_y[MAP ? 0 : i][wave][lane] = y;
    };
    const bool without = !ALL && n0 + NPT > N && __builtin_amdgcn_readfirstlane(s_odd[turn]) != 0;
    if (!ALL && tid == 0) s_odd[turn ^ 1] = 0;  // read before the last barrier, set after the next one
    if (!without && (MAP || (at.s >= 0 && at.end - tc >= len))) {  // no sequence ends within the chunk, but for its last token
      if (len == kTok) {
#pragma unroll
        for (int i = 0; i < kTok; ++i) step(i);
      } else {
        for (int i = 0; i < len; ++i) step(i);
      }
      if (!MAP && at.s < S && at.end == tc + len) end_state(at.s);
    } else {
      for (int i = 0; i < len; ++i) {
        const int t = tc + i;
        if (t >= at.end) {
          at.next(g.starts, t);
          if (at.s < S) begin_state(at.s);
        }
        if (without)
          step_without(i);
        else
          step(i);
        if (at.has(g.starts) && t == at.end - 1) end_state(at.s);
      }
    }
    __syncthreads();
    if (!MAP) {
#pragma unroll
      for (int k = 0; k < kOwn; ++k) {
        const int i = wave + 4 * k;
        const int64_t t = tc + i;
        if (i < len && act) {
          const float y = (s_y[i][0][lane] + s_y[i][1][lane]) + (s_y[i][2][lane] + s_y[i][3][lane]);
          const bool has = t >= first && t < last;
          const float o = fmaf(dp, o_u[k], y) * (o_z[k] * sigmoid_fast(o_z[k]));
          ((T*)g.out)[t * g.D + d] = from_f32<T>(has ? o : 0.0f);
        }
      }
    }
  };
  if (t0 < t1) {
    Chunk even, odd;
    load(even, t0);
    load(odd, t0 + kTok);
    if (!ALL) {
      if (tid < 2) s_odd[tid] = 0;
      __syncthreads();
    }
    for (int tc = t0; tc < t1; tc += 2 * kTok) {
      chunk(even, tc, 0);
      if (tc + kTok < t1) chunk(odd, tc + kTok, 1);
    }
  }
  if (MAP) {
    float* sums = &s_sc[0][0].x;
    __syncthreads();
    sums[tid] = sum;
    __syncthreads();
    if (wave == 0 && act) g.maps[seg * g.D + d] = whole ? (sums[lane] + sums[64 + lane]) + (sums[128 + lane] + sums[192 + lane]) : -1.0f;
    float* to = g.maps + g.segs * g.D + seg * N * g.D;
#pragma unroll
    for (int j = 0; j < NPT; ++j)
      if (act && n0 + j < N) to[(n0 + j) * g.D + d] = h[j];
  }
}

// The states that enter the segments: the state that segment k - 1 leaves replaces its map's. A workgroup has 64 states of a channel each,
// a lane each; its waves take the segments in chunks of kAhead, whose maps are all loaded at once: compose the chunk's from a zero state,
// take what enters it from the waves before, and go through it again. Segments that no sequence leaves have no map; what stands in
// its place is not used. (One lane a state and the segments one after another: 31 us for 256 of them, for the loads' latency.)
constexpr int kMaxSegs = 256, kAhead = 32, kJoinWaves = kMaxSegs / kAhead;
__global__ void __launch_bounds__(64 * kJoinWaves) join_kernel(ScanArgs g) {
  __shared__ float s_sum[kJoinWaves][64], s_end[kJoinWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t i = (int64_t)blockIdx.x * 64 + lane;
  const bool in = i < g.D * g.N;
  const int64_t d = in ? i % g.D : 0, n = in ? i / g.D : 0;
  const float a = g.A[d * g.N + n] * kLog2e;
  float* state = g.maps + g.segs * g.D + n * g.D + d;
  float S[kAhead], e[kAhead];
#pragma unroll
  for (int q = 0; q < kAhead; ++q) {
    const int64_t k = wave * kAhead + q;
    const bool has = k + 1 < g.segs;
    S[q] = has ? g.maps[k * g.D + d] : 0.0f;
    e[q] = has ? state[k * g.N * g.D] : 0.0f;
  }
  // x decayed over a sum of delta; in two parts: the factor may lie outside fp32 where its product with the state does not
  auto decayed = [&](float s, float x) __attribute__((always_inline)) {
    const float p = a * s, p0 = fminf(fmaxf(p, -126.0f), 127.0f), p1 = fminf(fmaxf(p - p0, -126.0f), 127.0f);
    return fast_exp2(p0) * (x * fast_exp2(p1));
  };
  float x = 0.0f, sum = 0.0f;
#pragma unroll
  for (int q = 0; q < kAhead; ++q) {
    x = S[q] < 0.0f ? e[q] : decayed(S[q], x) + e[q];
    sum = S[q] < 0.0f || sum < 0.0f ? -1.0f : sum + S[q];
  }
  s_sum[wave][lane] = sum;
  s_end[wave][lane] = x;
  __syncthreads();
  x = 0.0f;
  for (int w = 0; w < wave; ++w) x = s_sum[w][lane] < 0.0f ? s_end[w][lane] : decayed(s_sum[w][lane], x) + s_end[w][lane];
#pragma unroll
  for (int q = 0; q < kAhead; ++q) {
    const int64_t k = wave * kAhead + q;
    x = S[q] < 0.0f ? e[q] : decayed(S[q], x) + e[q];
    if (in && k + 1 < g.segs) state[k * g.N * g.D] = x;
  }
}

// ------------------------------------------------------------------------------------------ host
int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int64_t kMaxGrid = (1 << 24) - 1;
constexpr int kMaxN = 64;
constexpr int64_t kMaxTokens = 1 << 30;

int per_wave(int64_t N) { return N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : N <= 32 ? 8 : 16; }

// Tokens of a segment. A row that fills the chip is cut for six workgroups a CU (what LDS holds; 16384 x 1536 x 16 with four 229 us, with
// six 214), not below 64 tokens. A row that does not is latency, 0.15 us a token: segments of 32 (4096 x 256 x 16 with 256 tokens 84 us, 128
// 51, 64 34, 32 30), whole where the two passes more cost as much (77 tokens: 15 us whole).
int64_t segment_length(int64_t T, int64_t tiles) {
  if (T <= 128) return T > 0 ? T : 1;
  const int64_t cus = device_cus(), least = up(T, 32) * tiles <= 2 * cus ? 32 : 64;
  int64_t segs = up(6 * cus, tiles);
  if (segs > kMaxSegs) segs = kMaxSegs;
  const int64_t len = up(up(T, segs), kTok) * kTok;
  return len < least ? least : len;
}

int packed_status(int64_t T, int64_t S, int64_t D, int io) {
  if (T < 0 || S < 0 || D < 0 || (io != TSF_DTYPE_F32 && io != TSF_DTYPE_BF16)) return TSF_ERR_ARG;
  if (T > kMaxTokens || S > kMaxTokens || D > (int64_t)1 << 24) return TSF_ERR_UNSUPPORTED;
  return TSF_OK;
}

template <typename T, int RUN>
void launch_conv(ConvArgs a, int64_t K, hipStream_t st) {
  a.runs = up(a.starts.T, RUN);
  const unsigned grid = (unsigned)up((a.runs + a.starts.S) * a.groups, kThreads);
  switch (K) {
    case 2: conv_kernel<T, 2, RUN><<<grid, kThreads, 0, st>>>(a); break;
    case 3: conv_kernel<T, 3, RUN><<<grid, kThreads, 0, st>>>(a); break;
    case 4: conv_kernel<T, 4, RUN><<<grid, kThreads, 0, st>>>(a); break;
    case 5: conv_kernel<T, 5, RUN><<<grid, kThreads, 0, st>>>(a); break;
    case 6: conv_kernel<T, 6, RUN><<<grid, kThreads, 0, st>>>(a); break;
    case 7: conv_kernel<T, 7, RUN><<<grid, kThreads, 0, st>>>(a); break;
    default: conv_kernel<T, 8, RUN><<<grid, kThreads, 0, st>>>(a); break;
  }
}

template <typename T, int NPT, bool MAP>
void launch_scan(const ScanArgs& a, unsigned grid, hipStream_t st) {
  if (MAP || a.N == 4 * NPT)  // maps: states that do not exist go nowhere
    scan_kernel<T, NPT, MAP, true><<<grid, kThreads, 0, st>>>(a);
  else
    scan_kernel<T, NPT, false, false><<<grid, kThreads, 0, st>>>(a);
}
template <typename T, bool MAP>
void launch_scan(const ScanArgs& a, unsigned grid, hipStream_t st) {
  switch (per_wave(a.N)) {
    case 1: launch_scan<T, 1, MAP>(a, grid, st); break;
    case 2: launch_scan<T, 2, MAP>(a, grid, st); break;
    case 4: launch_scan<T, 4, MAP>(a, grid, st); break;
    case 8: launch_scan<T, 8, MAP>(a, grid, st); break;
    default: launch_scan<T, 16, MAP>(a, grid, st); break;
  }
}

// Tokens of a thread: four, which are done soonest (77 x 128 fp32 5 us, with sixteen 10; 65536 x 128 bf16 21 and 26), or sixteen, which read the
// taps and the rows before a run least often, where these are most, with 8 channels of bf16, and sixteen leave ten waves a CU or more (16384 x
// 1536 bf16 30 us, with four 37; fp32 48 and 44).
template <typename T>
void launch_conv(const ConvArgs& a, int64_t K, hipStream_t st) {
  if constexpr (sizeof(T) == 2) {
    if (up(a.starts.T, 16) * a.groups >= 640 * (int64_t)device_cus()) return launch_conv<T, 16>(a, K, st);
  }
  launch_conv<T, 4>(a, K, st);
}

int64_t conv_grid(int64_t T, int64_t S, int64_t D, int io) { return up((up(T, 4) + S) * up(D, io == TSF_DTYPE_BF16 ? 8 : 4), kThreads); }

}  // namespace

extern "C" {

int tsfast_hip_conv_packed(int64_t T, int64_t S, int64_t D, int64_t K, int io_dtype, int starts_int64, int weight_dtype, int bias_dtype,
                           const void* x, int64_t x_stride, const void* starts, const void* tails, const void* weight, const void* bias,
                           void* out, void* tails_out, void* stream) {
  const int rc = packed_status(T, S, D, io_dtype);
  if (rc != TSF_OK) return rc;
  if (K < 2) return TSF_ERR_ARG;
  if (K > kMaxK || conv_grid(T, S, D, io_dtype) > kMaxGrid) return TSF_ERR_UNSUPPORTED;
  if (D == 0 || (T == 0 && S == 0)) return TSF_OK;
  if (!starts || !weight || (T > 0 && (!x || !out || x_stride < 0)) || (S > 0 && !tails_out)) return TSF_ERR_ARG;
  ConvArgs a = {x, tails, weight, bias, out, tails_out, D, x_stride, up(D, io_dtype == TSF_DTYPE_BF16 ? 8 : 4), 0,
                Starts{starts, starts_int64, (int)S, (int)T}, weight_dtype == TSF_DTYPE_BF16, bias_dtype == TSF_DTYPE_BF16};
  if (io_dtype == TSF_DTYPE_BF16)
    launch_conv<bf16>(a, K, (hipStream_t)stream);
  else
    launch_conv<float>(a, K, (hipStream_t)stream);
  return tsf_launch_status();
}

int64_t tsfast_hip_mamba_packed_workspace_bytes(int64_t T, int64_t S, int64_t D, int64_t N) {
  if (packed_status(T, S, D, TSF_DTYPE_F32) != TSF_OK || N < 1 || N > kMaxN) return -1;
  if (D == 0 || T == 0) return 0;
  const int64_t segs = up(T, segment_length(T, up(D, kCh)));
  return segs > 1 ? segs * (N + 1) * D * 4 : 0;
}

int tsfast_hip_mamba_packed(int64_t T, int64_t S, int64_t D, int64_t N, int io_dtype, int starts_int64, const void* draw, int64_t draw_stride,
                            const float* A, const void* Bt, int64_t b_stride, const void* Ct, int64_t c_stride, const void* u,
                            int64_t u_stride, const void* z, int64_t z_stride, const float* Dp, const void* starts, const float* h0,
                            void* out, float* h_last, void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = packed_status(T, S, D, io_dtype);
  if (rc != TSF_OK) return rc;
  if (N < 1) return TSF_ERR_ARG;
  if (N > kMaxN) return TSF_ERR_UNSUPPORTED;
  if (D == 0 || (T == 0 && S == 0)) return TSF_OK;
  if (!A || !Dp || !starts || (S > 0 && !h_last)) return TSF_ERR_ARG;
  if (T > 0 && (!draw || !Bt || !Ct || !u || !z || !out)) return TSF_ERR_ARG;
  if (draw_stride < 0 || b_stride < 0 || c_stride < 0 || u_stride < 0 || z_stride < 0) return TSF_ERR_ARG;
  ScanArgs a = {draw, Bt, Ct, u, z, A, Dp, h0, out, h_last, draw_stride, b_stride, c_stride, u_stride, z_stride, D, up(D, kCh), 0, 1, (int)N,
                Starts{starts, starts_int64, (int)S, (int)T}, (float*)workspace};
  a.seg_len = segment_length(T, a.tiles);
  a.segs = T > 0 ? up(T, a.seg_len) : 1;
  if (a.segs * a.tiles > kMaxGrid) return TSF_ERR_UNSUPPORTED;
  const hipStream_t st = (hipStream_t)stream;
  if (a.segs > 1) {
    if (!workspace || workspace_bytes < tsfast_hip_mamba_packed_workspace_bytes(T, S, D, N)) return TSF_ERR_WORKSPACE;
    const unsigned grid = (unsigned)((a.segs - 1) * a.tiles);
    if (io_dtype == TSF_DTYPE_BF16)
      launch_scan<bf16, true>(a, grid, st);
    else
      launch_scan<float, true>(a, grid, st);
    join_kernel<<<(unsigned)up(D * N, 64), (unsigned)(64 * up(a.segs - 1, kAhead)), 0, st>>>(a);
  }
  const unsigned grid = (unsigned)(a.segs * a.tiles);
  if (io_dtype == TSF_DTYPE_BF16)
    launch_scan<bf16, false>(a, grid, st);
  else
    launch_scan<float, false>(a, grid, st);
  return tsf_launch_status();
}

}  // extern "C"
