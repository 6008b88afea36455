#pragma once
// Residual norm: the channel norm that closes a block, the block's gate and residual scale, the residual add and the channel norm that
// opens the next block, in one pass over the rows (gfx950, HBM-bound).  A row = the C channels of one position.
//
//   n = N_post(f)      rms: f r, r = 1 / sqrt(mean f^2 + eps);   layer: (f - mu) r, r = 1 / sqrt(mean (f - mu)^2 + eps);   none: f
//   y = x + s a(gate) (w n + b)          h = N_pre(y) w' + b'        (h from y before y is rounded)
// backward, from dy and dh, reads x, f and gate again and rebuilds y in fp32 -- the same bytes as reading y, and no rounding of y in the
// weight gradients:
//   t = dy + r' (dh w' - mean(dh w') - yhat mean(dh w' yhat))       dx = t
//   d = t s a w;   df = r (d - mean(d) - n mean(d n))                (rms: no mean(d), mean(dh w') terms)
//   dgate = s a' (w T1 + b T2) over the rows of a gate, T1 = sum t n, T2 = sum t;   with t1 = sum a T1, t2 = sum a T2 over the gates:
//   ds = w t1 + b t2,  dw = s t1,  db = s t2;   dw' = sum dh yhat,  db' = sum dh
// so two column sums carry the gradients of gate, scale, weight and bias.  No atomics: a block leaves one row of column sums per
// accumulator, a second launch adds the rows in a fixed order in 64 bits.
//
// A TEAM of lanes owns a row: 1 .. 64 lanes of a wave (sums by DPP), or the whole block (sums through LDS).  A lane holds NV x 8
// adjacent channels in registers, so a row is read once; the loads of a team's next row are in flight while it works on the current one.
// Accesses are 16 bytes at the alignment of an element (the memory path of gfx950 takes any), so odd widths and strides run the same
// code.
//
// What bounds it (a copy of 4 GB: 4.8 TB/s, 256 MB: 5.4): memory.  Counters give the bytes of the formula, for a backward pass the
// blocks' column sums besides (16384 x 4096: 8 MB of 1.49 GB).  Forward, 32768 x 2048,
// fp32 residual and bf16 branch, 805 MB: 146 us, 5.5 TB/s; 401408 x 64 bf16: 41 us, 5.0.  Backward, 401408 x 64: 308 MB in 64 us, 4.8 TB/s;
// 16384 x 4096, fp32 / bf16, a gate per element: 1.48 GB in 304 us, 4.9 TB/s.  The second launch of a backward pass: 6 - 20 us.
#include "common.h"
#include <hip/hip_fp16.h>
#include <atomic>

namespace {
__device__ __forceinline__ float h2f(uint16_t h) { return __half2float(__ushort_as_half(h)); }
__device__ __forceinline__ uint16_t f2h(float f) { return __half_as_ushort(__float2half_rn(f)); }
template <int T> __device__ __forceinline__ float ld1(const void* p, int64_t e) {
  if (T == MSCL_F32) return ((const float*)p)[e];
  const uint16_t h = ((const uint16_t*)p)[e];
  return T == MSCL_BF16 ? bf2f(h) : h2f(h);
}
template <int T> __device__ __forceinline__ void st1(void* p, int64_t e, float v) {
  if (T == MSCL_F32) ((float*)p)[e] = v;
  else ((uint16_t*)p)[e] = T == MSCL_BF16 ? f2bf(v) : f2h(v);
}

// 8 channels as they lie in memory
template <int T> struct Raw { uint32_t w[T == MSCL_F32 ? 8 : 4]; };
template <int T> __device__ __forceinline__ void unpack(const Raw<T>& u, float* v) {
  if (T == MSCL_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(u.w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = T == MSCL_BF16 ? __uint_as_float(u.w[i] << 16) : h2f((uint16_t)u.w[i]);
      v[2 * i + 1] = T == MSCL_BF16 ? __uint_as_float(u.w[i] & 0xFFFF0000u) : h2f((uint16_t)(u.w[i] >> 16));
    }
  }
}

// A lane's channels of a row: value (q, i) is channel col[q] + i, 8 adjacent ones.  The last vector of a row that is no multiple of 8 wide
// ends with the row, and so repeats up to 7 channels of the vector before it: both lanes compute -- and store -- the same bits for
// them, and the first `skip` values of the later one stay out of the row's sums.  A lane past the row repeats the last vector, skips all
// 8 and stores nothing.  So every load is one unconditional access of 16 (32) bytes.  NARROW: rows of fewer than 8 channels have
// their values at the end of one vector and go element by element.
template <int NV, bool NARROW> struct Cols {
  int col[NV], skip[NV];
  __device__ __forceinline__ Cols(int lane, int T, int C) {
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      const int at = (q * T + lane) * 8;
      skip[q] = at >= C ? 8 : at + 8 > C ? at + 8 - C : 0;
      col[q] = at + 8 > C ? C - 8 : at;
    }
  }
  template <int TY> __device__ __forceinline__ void fetch(const void* p, int64_t row, Raw<TY> (&u)[NV]) const {
    constexpr int sz = TY == MSCL_F32 ? 4 : 2;
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      const char* a = (const char*)p + (row + col[q]) * sz;
      if (!NARROW) {
        if (TY == MSCL_F32) __builtin_memcpy(u[q].w, (const float*)a, 32);
        else __builtin_memcpy(u[q].w, (const uint16_t*)a, 16);
      } else {
#pragma unroll
        for (int i = 0; i < (TY == MSCL_F32 ? 8 : 4); ++i) u[q].w[i] = 0;
#pragma unroll
        for (int i = 1; i < 8; ++i)
          if (i >= skip[q]) {
            if (TY == MSCL_F32) u[q].w[i] = ((const uint32_t*)a)[i];
            else u[q].w[i >> 1] |= (uint32_t)((const uint16_t*)a)[i] << (16 * (i & 1));
          }
      }
    }
  }
  template <int TY> __device__ __forceinline__ void load(const void* p, int64_t row, float (&v)[NV][8]) const {
    Raw<TY> u[NV];
    fetch<TY>(p, row, u);
#pragma unroll
    for (int q = 0; q < NV; ++q) unpack<TY>(u[q], v[q]);
  }
  // a per-channel vector; a missing one is all `one`
  __device__ __forceinline__ void load_vec(const float* p, float one, float (&v)[NV][8]) const {
    if (p) load<MSCL_F32>(p, 0, v);
    else
#pragma unroll
      for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[q][i] = one;
  }
  template <int TY> __device__ __forceinline__ void store(void* p, int64_t row, const float (&v)[NV][8]) const {
    constexpr int sz = TY == MSCL_F32 ? 4 : 2;
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      char* a = (char*)p + (row + col[q]) * sz;
      if (skip[q] == 8) continue;
      if (!NARROW) {
        if (TY == MSCL_F32) __builtin_memcpy((float*)a, v[q], 32);
        else {
          uint32_t w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            w[i] = TY == MSCL_BF16 ? pack2bf(v[q][2 * i], v[q][2 * i + 1]) : (uint32_t)f2h(v[q][2 * i]) | (uint32_t)f2h(v[q][2 * i + 1]) << 16;
          __builtin_memcpy((uint16_t*)a, w, 16);
        }
      } else {
#pragma unroll
        for (int i = 1; i < 8; ++i) if (i >= skip[q]) st1<TY>(a, i, v[q][i]);
      }
    }
  }
  // sum of f(q, i) over the lane's own channels
  template <class F> __device__ __forceinline__ float sum(F f) const {
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) t += f(q, i);
      if (skip[q]) {
        t = 0.f;
#pragma unroll
        for (int i = 1; i < 8; ++i) t += i >= skip[q] ? f(q, i) : 0.f;
      }
      s += t;
    }
    return s;
  }
};

// team sums.  WAVE: T in {1, 2, 4, 8, 16, 32, 64}.  Block teams: waves meet in LDS; two alternating slots make one barrier per sum enough
// (a slot is written again only by waves that have passed the barrier of the sum between, i.e. after every wave has read it).
template <int CTRL> __device__ __forceinline__ float dpp_add(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}
// A row of 16 lanes to one value, the same bits in each of them: every step adds the two halves of a pair in both halves (half mirror: the
// other quad of 8 lanes), and an addition commutes.  A rotation by a quad would add four quads in two different orders, and the lanes that
// share a channel would store different bits for it (9 waves or more: the last bit of 1 / deviation in a tenth of the rows).
__device__ __forceinline__ float row16_same(float v) {
  return dpp_add<0x128>(dpp_add<0x141>(dpp_add<0x4E>(dpp_add<0xB1>(v))));
}
template <bool WAVE> struct Team {
  int T;
  float2* red;          // block teams: [2][16]
  int slot;
  __device__ __forceinline__ float wsum(float v) const {
    if (T == 64) return wave_sum(v);
    if (T >= 2) v = dpp_add<0xB1>(v);        // quad_perm: neighbour
    if (T >= 4) v = dpp_add<0x4E>(v);        // quad_perm: other pair
    if (T >= 8) v = dpp_add<0x141>(v);       // row_half_mirror: other quad
    if (T >= 16) v = dpp_add<0x128>(v);      // row_ror 8: other half row
    if (T == 32) {                           // the rows of a pair: {r0, r0, r2, r2} + {r1, r1, r3, r3}
      const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
      v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    }
    return v;
  }
  __device__ __forceinline__ float2 sum2(float a, float b, bool want_b) {
    if (WAVE) return make_float2(wsum(a), want_b ? wsum(b) : 0.f);
    a = wave_sum(a);
    if (want_b) b = wave_sum(b);
    const int w = threadIdx.x >> 6, nw = blockDim.x >> 6, l = threadIdx.x & 15;
    float2* s = red + slot * 16;
    slot ^= 1;
    if ((threadIdx.x & 63) == 0) s[w] = make_float2(a, b);
    __syncthreads();
    const float2 t = l < nw ? s[l] : make_float2(0.f, 0.f);          // every 16 lanes add the (at most 16) waves' values
    return make_float2(row16_same(t.x), want_b ? row16_same(t.y) : 0.f);
  }
  __device__ __forceinline__ float sum(float a) { return sum2(a, 0.f, false).x; }
};

// exp(x) for x <= 0 to about 2 ulp: the rounding of x log2(e) is put back to first order.  It is 0 from -104 on (and flushed below 2^-126), so
// -150 stands for all that is lower: a shut gate has the type's lowest value or -inf, whose product overflows and leaves no correction.  (Not
// fmaxf, which would take a NaN for a shut gate.)
__device__ __forceinline__ float exp_neg(float x) {
  x = x < -150.f ? -150.f : x;
  const float t = x * 1.44269504f, lo = fmaf(x, 1.92596303e-8f, fmaf(x, 1.44269504f, -t));
  const float e = __builtin_amdgcn_exp2f(t);
  return fmaf(e, lo * 0.693147181f, e);
}
// gate value a(g) and slope a'(g).  With e = exp(-|g|), q = 1 / (1 + e): sigmoid is q or e q by the sign of g, its slope e q^2; tanh's slope
// 4 e q^2 with e = exp(-2 |g|).  No difference of near numbers, which a (1 - a) and 1 - a^2 are for a saturated gate.  (q: the 1-ulp reciprocal.)
__device__ __forceinline__ float2 act_both(int act, float g) {
  if (act == MSCL_GATE_SIGMOID) {
    const float e = exp_neg(-fabsf(g)), q = __builtin_amdgcn_rcpf(1.f + e), eq = e * q;
    return make_float2(g >= 0.f ? q : eq, eq * q);
  }
  if (act == MSCL_GATE_TANH) {
    const float e = exp_neg(-2.f * fabsf(g)), q = __builtin_amdgcn_rcpf(1.f + e);
    return make_float2(tanhf(g), 4.f * e * q * q);
  }
  return make_float2(g, 1.f);
}
// the values (and slopes) of a lane's gates, one branch for all of them
template <bool SLOPE, int NV>
__device__ __forceinline__ void act_row(int act, float (&a)[NV][8], float (*slope)[8]) {
  auto each = [&](int kind) {
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float2 v = act_both(kind, a[q][i]);
        a[q][i] = v.x;
        if (SLOPE) slope[q][i] = v.y;
      }
  };
  if (act == MSCL_GATE_SIGMOID) each(MSCL_GATE_SIGMOID);
  else if (act == MSCL_GATE_TANH) each(MSCL_GATE_TANH);
  else each(MSCL_GATE_LINEAR);
}

#define EACH _Pragma("unroll") for (int q = 0; q < NV; ++q) _Pragma("unroll") for (int i = 0; i < 8; ++i)

// mean and 1 / deviation of a row held in v (rms: mean 0); the second moment is taken about the mean, in a second pass over registers
template <int NV, bool WAVE, class C>
__device__ __forceinline__ float2 row_stats(const float (&v)[NV][8], int kind, float inv_c, float eps, const C& c, Team<WAVE>& team) {
  float mu = 0.f;
  if (kind == MSCL_NORM_LAYER) mu = team.sum(c.sum([&](int q, int i) { return v[q][i]; })) * inv_c;
  const float s = c.sum([&](int q, int i) { const float d = v[q][i] - mu; return d * d; });
  return make_float2(mu, 1.f / sqrtf(team.sum(s) * inv_c + eps));
}
}  // namespace

// A block takes `share` consecutive rows, its teams in turn.  EACH_GATE: a gate for every row, fetched with it; otherwise the gate's
// activation stays in registers until a row belongs to another gate.  BIAS: b_post or b_pre present.
template <int XT, int FT, int NV, bool WAVE, bool EACH_GATE, bool BIAS, bool NARROW>
__global__ __launch_bounds__(WAVE ? 256 : 1024) void res_norm_fwd_kernel(mscl_res_norm_desc d, int T, FastDiv gdiv, int64_t share) {
  __shared__ float2 red[32];
  Team<WAVE> team{T, red, 0};
  const int per = WAVE ? 256 / T : 1, sub = WAVE ? (int)threadIdx.x / T : 0;
  const int lane = WAVE ? (int)threadIdx.x % T : (int)threadIdx.x;
  const Cols<NV, NARROW> c(lane, T, d.C);
  const float inv_c = 1.f / (float)d.C;
  const int64_t end = share * (blockIdx.x + 1) < d.rows ? share * (blockIdx.x + 1) : d.rows;
  int64_t r = share * blockIdx.x + sub;
  Raw<XT> ux[NV];
  Raw<FT> uf[NV], ug[NV];
  constexpr bool LEAN = NV > 1;
  auto fetch = [&](int64_t at) {
    c.template fetch<XT>(d.x, at * d.ld_x, ux);
    if (d.f) c.template fetch<FT>(d.f, at * d.ld_f, uf);
    if (EACH_GATE) c.template fetch<FT>(d.gate, at * d.C, ug);
  };
  if (!LEAN && r < end) fetch(r);
  float sw[NV][8], sb[BIAS ? NV : 1][8], w2[NV][8], b2[BIAS ? NV : 1][8], a[NV][8];
  auto post_vectors = [&] {
    float s[NV][8];
    c.load_vec(d.scale, 1.f, s);
    c.load_vec(d.w_post, 1.f, sw);
    EACH sw[q][i] *= s[q][i];
    if constexpr (BIAS) {
      c.load_vec(d.b_post, 0.f, sb);
      EACH sb[q][i] *= s[q][i];
    }
  };
  auto pre_vectors = [&] {
    c.load_vec(d.w_pre, 1.f, w2);
    if constexpr (BIAS) c.load_vec(d.b_pre, 0.f, b2);
  };
  if (!LEAN && d.f) post_vectors();
  if (!LEAN && d.pre) pre_vectors();
  EACH a[q][i] = 1.f;
  int gate = -1;
  for (; r < end; r += per) {
    float x[NV][8], f[NV][8];
    if (LEAN) fetch(r);
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      unpack<XT>(ux[q], x[q]);
      if (d.f) unpack<FT>(uf[q], f[q]);
      if (EACH_GATE) unpack<FT>(ug[q], a[q]);
    }
    if (!LEAN && r + per < end) fetch(r + per);
    if (d.f) {
      if (EACH_GATE) {
        act_row<false, NV>(d.gate_act, a, nullptr);
      } else if (d.gate) {
        const int g = d.rows_per_gate < d.rows ? fdiv((int)r, gdiv) : 0;
        if (g != gate) {
          gate = g;
          c.template load<FT>(d.gate, (int64_t)g * d.C, a);
          act_row<false, NV>(d.gate_act, a, nullptr);
        }
      }
      if (d.post) {
        const float2 st = row_stats<NV, WAVE>(f, d.post, inv_c, d.eps, c, team);
        if (lane == 0) {
          if (d.mean_f) d.mean_f[r] = st.x;
          if (d.rstd_f) d.rstd_f[r] = st.y;
        }
        EACH f[q][i] = (f[q][i] - st.x) * st.y;
      }
      if (LEAN) post_vectors();
      EACH x[q][i] += a[q][i] * (BIAS ? sw[q][i] * f[q][i] + sb[BIAS ? q : 0][i] : sw[q][i] * f[q][i]);
      c.template store<XT>(d.y, r * d.C, x);
    }
    if (d.pre) {
      const float2 st = row_stats<NV, WAVE>(x, d.pre, inv_c, d.eps, c, team);
      if (lane == 0) {
        if (d.mean_y) d.mean_y[r] = st.x;
        if (d.rstd_y) d.rstd_y[r] = st.y;
      }
      if (LEAN) pre_vectors();
      EACH { x[q][i] = (x[q][i] - st.x) * st.y * w2[q][i]; if (BIAS) x[q][i] += b2[BIAS ? q : 0][i]; }
      c.template store<FT>(d.h, r * d.C, x);
    }
  }
}

// Which rows a block of the backward pass takes, and which column sums it leaves.
//   SPLIT  the gates are long runs of rows (or there is one, or none): `per_gate` blocks share the rows of a gate, their T1 / T2 stay
//          apart per gate until the second launch has added them up and applied a and a'
//   WHOLE  the gates are short or very many: a team takes whole gates, applies a itself and writes dgate at the end of each
//   EACH1  a gate for every row: as WHOLE with runs of one row, and nothing to keep between rows but the totals
enum { SPLIT = 0, WHOLE = 1, EACH1 = 2 };
struct BwdPlan { int T, wave, nv, mode, per_gate, gates, blocks, rows_per_gate, share; };

// Waves a SIMD of the backward kernel (512 registers a lane shared among them): 3, which most forms run in without spills (a training pass of
// 24 M elements, C = 192: bf16 110 us at 4, 108 at 3; fp32 290 at 4, 206 at 3), 2 for those with more sums (a gate per element and biases,
// C = 192: bf16 144 us at 3, 141 at 2; fp32 422 at 3, 253 at 2; fp32 / bf16 in whole gates of 8 rows 221 and 167; bf16 in whole gates 130 at 3, 143 at
// 2).  A gate per element without biases takes what it needs by itself (5856 x 4096 bf16: 127 us, 143 when told 3).  More than 768 lanes: 4.
// LEAN (past 8192 channels, 16 of them a lane, 1024 lanes): no prefetch, the per-channel vectors read again for every row -- registers.  LAZY: each
// where it is used (2000 x 12000, a training pass: bf16 313 -> 276 us, fp32 / bf16 392 -> 300; whole gates lose, 467 -> 567).
// LATE (also most forms of more than 768 lanes): a row's loads begin with its work (2928 x 8192, a training pass: fp32 with a gate per element 374
// us with the next row in flight and spills, 259 without; bf16, no gate, no spills, 107 and 112).
constexpr int bwd_waves(int threads, int xt, int ft, int mode, bool bias) {
  return threads > 768 ? 4 : threads <= 512 && ((mode == EACH1 && (ft == MSCL_F32 || bias)) || (mode == WHOLE && xt == MSCL_F32)) ? 2 : 3;
}
// Column sums that the backward kernel keeps in LDS: all four, two where 16 channels a lane and biases would need 256 KB.  (2928 x 8192, a training
// pass, in registers with spills and so: bf16 with biases 181 / 117 us, with a gate per element as well 285 / 182; 4800 x 5000 fp32, a gate per
// element and biases 377 / 268, bf16 164 / 160, without gates 130 / 134.)
constexpr int bwd_in_lds(int nv, int threads, int xt, int mode, bool bias) {
  return threads > 768 ? (nv == 2 && bias ? 2 : 4) : threads > 512 && xt == MSCL_F32 && mode != SPLIT && bias ? 4 : 0;
}
template <int K> struct Sum { static constexpr int value = K; };
template <int XT, int FT, int NV, bool WAVE, int THREADS, int MODE, bool BIAS, bool NARROW>
__global__ __launch_bounds__(THREADS, THREADS <= 512 && MODE == EACH1 && !BIAS ? 1 : bwd_waves(THREADS, XT, FT, MODE, BIAS)) void res_norm_bwd_kernel(mscl_res_norm_desc d, BwdPlan pl) {
  extern __shared__ float lds[];                    // wave teams: [256][8 NV] for the column sums of a block; bwd_in_lds: held()
  __shared__ float2 red[32];
  constexpr int NB = BIAS ? NV : 1;
  const int T = pl.T;
  Team<WAVE> team{T, red, 0};
  const int per = WAVE ? 256 / T : 1, sub = WAVE ? (int)threadIdx.x / T : 0;
  const int lane = WAVE ? (int)threadIdx.x % T : (int)threadIdx.x;
  const Cols<NV, NARROW> c(lane, T, d.C);
  const float inv_c = 1.f / (float)d.C;
  const bool layer2 = d.pre == MSCL_NORM_LAYER, layer1 = d.post == MSCL_NORM_LAYER;

  // the team's rows: r, r + step, ... < end; WHOLE: runs of rows_per_gate rows
  int64_t r, step, end, gate = 0;
  if (MODE == SPLIT) {
    const int64_t g = blockIdx.x / pl.per_gate, j = blockIdx.x % pl.per_gate;
    const int64_t share = pl.share, r0 = g * pl.rows_per_gate;
    end = r0 + (share * (j + 1) < pl.rows_per_gate ? share * (j + 1) : pl.rows_per_gate);
    r = r0 + share * j + sub;
    step = per;
    gate = g;
  } else {
    gate = (int64_t)blockIdx.x * per + sub;
    step = (int64_t)gridDim.x * per;                // in gates
    r = gate * pl.rows_per_gate;
    end = d.rows;
  }
  auto after = [&](int64_t at) {
    if (MODE != WHOLE) return at + step;
    return (at + 1) % pl.rows_per_gate ? at + 1 : at + 1 + (step - 1) * pl.rows_per_gate;
  };
  Raw<XT> ux[NV], uy[NV];
  Raw<FT> uf[NV], uh[NV], ug[NV];
  float sd[4] = {0.f, 1.f, 0.f, 1.f};               // mean_f, rstd_f, mean_y, rstd_y of the row that is on its way
  auto fetch = [&](int64_t at) {
    c.template fetch<XT>(d.x, at * d.ld_x, ux);
    if (d.f) c.template fetch<FT>(d.f, at * d.ld_f, uf);
    if (d.dy) c.template fetch<XT>(d.dy, at * d.C, uy);
    if (d.dh) c.template fetch<FT>(d.dh, at * d.C, uh);
    if (MODE == EACH1) c.template fetch<FT>(d.gate, at * d.C, ug);
    if (d.f && d.post) { if (layer1) sd[0] = d.mean_f[at]; sd[1] = d.rstd_f[at]; }
    if (d.dh) { if (layer2) sd[2] = d.mean_y[at]; sd[3] = d.rstd_y[at]; }
  };
  constexpr bool LEAN = NV > 1, LAZY = LEAN && MODE != WHOLE, LATE = LEAN || (THREADS > 768 && !(MODE == SPLIT && (!BIAS || XT != MSCL_F32)));
  if (!LATE && r < end) fetch(r);

  float sw[NV][8], sb[NB][8], w2[NV][8], a[NV][8];
  float U1[NV][8] = {}, U2[NB][8] = {}, T1[NV][8] = {}, T2[NB][8] = {}, t1[MODE == WHOLE ? NV : 1][8] = {}, t2[MODE == WHOLE ? NB : 1][8] = {};
  auto post_vectors = [&] {
    if (LAZY) asm volatile("" ::: "memory");         // not before the values of the step above are done with
    float s[NV][8];
    c.load_vec(d.scale, 1.f, s);
    c.load_vec(d.w_post, 1.f, sw);
    EACH sw[q][i] *= s[q][i];
    if constexpr (BIAS) {
      c.load_vec(d.b_post, 0.f, sb);
      EACH sb[q][i] *= s[q][i];
    }
  };
  auto pre_vectors = [&] {
    if (LAZY) asm volatile("" ::: "memory");
    c.load_vec(d.w_pre, 1.f, w2);
  };
  if (!LEAN && d.f) post_vectors();
  if (!LEAN && d.dh) pre_vectors();
  EACH a[q][i] = 1.f;
  if (MODE == SPLIT && d.gate) {
    c.template load<FT>(d.gate, gate * d.C, a);
    act_row<false, NV>(d.gate_act, a, nullptr);
  }
  int64_t loaded = -1;

  // Column sum K += f.  Where registers lack (bwd_in_lds) the sums K < IN_LDS live in LDS, 16 bytes a lane at a time.
  constexpr int IN_LDS = bwd_in_lds(NV, THREADS, XT, MODE, BIAS);
  auto held = [&](int k, int q, int h) -> float4& { return ((float4*)lds)[(((BIAS ? k : k / 2) * NV + q) * 2 + h) * T + lane]; };
  auto add = [&](auto K, auto& sum, auto f) {
    if constexpr (K.value < IN_LDS) {
#pragma unroll
      for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float4 v = held(K.value, q, h);
          v.x += f(q, 4 * h); v.y += f(q, 4 * h + 1); v.z += f(q, 4 * h + 2); v.w += f(q, 4 * h + 3);
          held(K.value, q, h) = v;
        }
    } else EACH sum[q][i] += f(q, i);
  };
  if (IN_LDS)
    for (int k = 0; k < IN_LDS; k += BIAS ? 1 : 2)
      for (int j = 0; j < 2 * NV; ++j) held(k, j / 2, j % 2) = make_float4(0.f, 0.f, 0.f, 0.f);         // a lane's own, no barrier

  while (r < end) {
    float x[NV][8], n[NV][8], t[NV][8], g[NV][8];
    if (LATE) fetch(r);
    if (LEAN && !LAZY) { if (d.f) post_vectors(); if (d.dh) pre_vectors(); }
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      unpack<XT>(ux[q], x[q]);
      if (d.f) unpack<FT>(uf[q], n[q]);
      if (d.dy) unpack<XT>(uy[q], t[q]);
      if (d.dh) unpack<FT>(uh[q], g[q]);
      if (MODE == EACH1) unpack<FT>(ug[q], a[q]);
    }
    const float mu1 = sd[0], r1 = sd[1], mu2 = sd[2], r2 = sd[3];
    const int64_t next = after(r);
    if (!LATE && next < end) fetch(next);
    if (!d.dy) EACH t[q][i] = 0.f;
    float slope[MODE == EACH1 ? NV : 1][8];
    if constexpr (MODE == EACH1) {
      act_row<true, NV>(d.gate_act, a, slope);
    }
    if constexpr (MODE == WHOLE) {
      if (gate != loaded) {
        loaded = gate;
        c.template load<FT>(d.gate, gate * d.C, a);
        act_row<false, NV>(d.gate_act, a, nullptr);
      }
    }
    if (d.f) {
      if (d.post) EACH n[q][i] = (n[q][i] - mu1) * r1;
      if (LAZY && d.dh) post_vectors();
      if (d.dh) EACH x[q][i] += a[q][i] * (BIAS ? sw[q][i] * n[q][i] + sb[BIAS ? q : 0][i] : sw[q][i] * n[q][i]);        // y
    }
    if (d.dh) {
      EACH x[q][i] = (x[q][i] - mu2) * r2;          // yhat
      add(Sum<0>(), U1, [&](int q, int i) { return g[q][i] * x[q][i]; });
      if constexpr (BIAS) add(Sum<1>(), U2, [&](int q, int i) { return g[q][i]; });
      if (LAZY) pre_vectors();
      EACH g[q][i] *= w2[q][i];
      const float c1 = c.sum([&](int q, int i) { return g[q][i] * x[q][i]; });
      const float c0 = layer2 ? c.sum([&](int q, int i) { return g[q][i]; }) : 0.f;
      const float2 s = team.sum2(c1, c0, layer2);
      const float m1 = s.x * inv_c, m0 = s.y * inv_c;
      EACH t[q][i] += r2 * (g[q][i] - m0 - x[q][i] * m1);
    }
    if (d.dx) c.template store<XT>(d.dx, r * d.C, t);
    if (d.f) {
      if (LAZY) post_vectors();
      if constexpr (MODE == EACH1) {
        add(Sum<2>(), T1, [&](int q, int i) { return a[q][i] * (t[q][i] * n[q][i]); });
        if constexpr (BIAS) add(Sum<3>(), T2, [&](int q, int i) { return a[q][i] * t[q][i]; });
        EACH slope[q][i] *= BIAS ? sw[q][i] * (t[q][i] * n[q][i]) + sb[BIAS ? q : 0][i] * t[q][i] : sw[q][i] * (t[q][i] * n[q][i]);
      } else if constexpr (MODE == SPLIT) {
        add(Sum<2>(), T1, [&](int q, int i) { return t[q][i] * n[q][i]; });
        if constexpr (BIAS) add(Sum<3>(), T2, [&](int q, int i) { return t[q][i]; });
      } else {
        EACH { T1[q][i] += t[q][i] * n[q][i]; T2[BIAS ? q : 0][i] += t[q][i]; }
      }
      EACH t[q][i] = t[q][i] * a[q][i] * sw[q][i];
      if constexpr (MODE == EACH1) { if (d.dgate) c.template store<FT>(d.dgate, r * d.C, slope); }
      if (d.df) {
        if (d.post) {
          const float k1 = c.sum([&](int q, int i) { return t[q][i] * n[q][i]; });
          const float k0 = layer1 ? c.sum([&](int q, int i) { return t[q][i]; }) : 0.f;
          const float2 s = team.sum2(k1, k0, layer1);
          const float m1 = s.x * inv_c, m0 = s.y * inv_c;
          EACH t[q][i] = r1 * (t[q][i] - m0 - n[q][i] * m1);
        }
        c.template store<FT>(d.df, r * d.C, t);
      }
      if constexpr (MODE == WHOLE) {
        if (next != r + 1 || next >= end || pl.rows_per_gate == 1) {        // the gate's last row
          c.template load<FT>(d.gate, gate * d.C, x);
          act_row<true, NV>(d.gate_act, x, n);
          add(Sum<2>(), t1, [&](int q, int i) { return a[q][i] * T1[q][i]; });
          add(Sum<3>(), t2, [&](int q, int i) { return a[q][i] * T2[BIAS ? q : 0][i]; });
          EACH {
            x[q][i] = n[q][i] * (sw[q][i] * T1[q][i] + sb[BIAS ? q : 0][i] * T2[BIAS ? q : 0][i]);
            T1[q][i] = T2[BIAS ? q : 0][i] = 0.f;
          }
          if (d.dgate) c.template store<FT>(d.dgate, gate * d.C, x);
          gate += step;
        }
      }
    }
    r = next;
  }

  // the block's column sums: [4][C] floats (U1, U2, T1, T2; with the gates applied: t1, t2 in the place of T1, T2)
  float* out = d.ws + (int64_t)blockIdx.x * 4 * d.C;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (!BIAS && (k & 1)) continue;
    if (k < 2 ? !d.dh : !d.f) continue;             // block-uniform
    float v[NV][8];
    if (k < IN_LDS) {
#pragma unroll
      for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float4 u = held(k, q, h);
          v[q][4 * h] = u.x; v[q][4 * h + 1] = u.y; v[q][4 * h + 2] = u.z; v[q][4 * h + 3] = u.w;
        }
    } else
      EACH v[q][i] = k == 0 ? U1[q][i] : k == 1 ? U2[BIAS ? q : 0][i] : k == 2 ? (MODE == WHOLE ? t1[MODE == WHOLE ? q : 0][i] : T1[q][i])
                 : (MODE == WHOLE ? t2[MODE == WHOLE && BIAS ? q : 0][i] : T2[BIAS ? q : 0][i]);
    if (!WAVE) { c.template store<MSCL_F32>(out + (int64_t)k * d.C, 0, v); continue; }
    __syncthreads();
    EACH if (i >= c.skip[q]) lds[sub * T * 8 * NV + c.col[q] + i] = v[q][i];
    __syncthreads();
    for (int e = threadIdx.x; e < d.C; e += 256) {
      float s = 0.f;
      for (int u = 0; u < per; ++u) s += lds[u * T * 8 * NV + e];
      out[(int64_t)k * d.C + e] = s;
    }
  }
}
#undef EACH

// Adds the blocks' column sums: COLS columns x 512 / COLS lanes per block, in 64 bits and in a fixed order.  Split gates: lanes_per_gate
// lanes share the blocks of a gate, the first of them writes dgate and goes on with a T1, a T2.  The launch is latency alone, so a lane
// has AT_ONCE loads of a sum in flight (out of range: the last row again, times zero), and narrow rows spread over more blocks (COLS 4).
template <int FT, int COLS>
__global__ __launch_bounds__(512) void res_norm_finish_kernel(mscl_res_norm_desc d, BwdPlan pl, int lanes_per_gate) {
  constexpr int AT_ONCE = 8, LANES = 512 / COLS, IN_WAVE = 64 / COLS;
  __shared__ double red[4][LANES][COLS];
  const int cl = threadIdx.x % COLS, lane = threadIdx.x / COLS;
  const int col = blockIdx.x * COLS + cl, C = d.C, at = col < C ? col : C - 1;        // columns past C compute the last one and drop it
  const bool in = col < C, split = pl.mode == SPLIT && d.gate;
  const int64_t stride = (int64_t)4 * C;
  double v[4] = {0.0, 0.0, 0.0, 0.0};
  // rows first, first + hop, ... below `rows` of sum k
  auto add = [&](int k, int64_t row0, int first, int hop, int rows) {
    double s = 0.0;
    const float* p = d.ws + row0 * stride + (int64_t)k * C + at;
    for (int b = first; b < rows; b += hop * AT_ONCE) {
      float x[AT_ONCE];
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) { const int e = b + hop * j; x[j] = p[(e < rows ? e : rows - 1) * stride]; }
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) s += b + hop * j < rows ? (double)x[j] : 0.0;
    }
    return s;
  };
  if (d.dh) {
    v[0] = add(0, 0, lane, LANES, pl.blocks);
    if (d.db_pre) v[1] = add(1, 0, lane, LANES, pl.blocks);
  }
  const double w = d.w_post ? (double)d.w_post[at] : 1.0, b = d.b_post ? (double)d.b_post[at] : 0.0;
  const double s = d.scale ? (double)d.scale[at] : 1.0;
  if (d.f && !split) {
    v[2] = add(2, 0, lane, LANES, pl.blocks);
    if (d.b_post) v[3] = add(3, 0, lane, LANES, pl.blocks);
  } else if (split) {
    const int at_once = LANES / lanes_per_gate, mine = lane / lanes_per_gate, part = lane % lanes_per_gate;
    for (int g0 = 0; g0 < pl.gates; g0 += at_once) {
      const int g = g0 + mine;
      double s1 = 0.0, s2 = 0.0;
      float logit = 0.f;
      if (g < pl.gates) {
        logit = ld1<FT>(d.gate, (int64_t)g * C + at);
        s1 = add(2, (int64_t)g * pl.per_gate, part, lanes_per_gate, pl.per_gate);
        if (d.b_post) s2 = add(3, (int64_t)g * pl.per_gate, part, lanes_per_gate, pl.per_gate);
      }
      if (lanes_per_gate > 1) {
        __syncthreads();
        red[0][lane][cl] = s1;
        red[1][lane][cl] = s2;
        __syncthreads();
        if (part == 0)
          for (int i = 1; i < lanes_per_gate; ++i) { s1 += red[0][lane + i][cl]; s2 += red[1][lane + i][cl]; }
      }
      if (part == 0 && g < pl.gates) {
        const float2 a = act_both(d.gate_act, logit);
        v[2] += (double)a.x * s1;
        v[3] += (double)a.x * s2;
        if (d.dgate && in) st1<FT>(d.dgate, (int64_t)g * C + col, (float)(s * (double)a.y * (w * s1 + b * s2)));
      }
    }
    __syncthreads();
  }
  // over the lanes of a column: those of a wave, then the waves through LDS
#pragma unroll
  for (int k = 0; k < 4; ++k) {
#pragma unroll
    for (int o = COLS; o < 64; o <<= 1) v[k] += __shfl_xor(v[k], o, 64);
    if (lane % IN_WAVE == 0) red[k][lane / IN_WAVE][cl] = v[k];
  }
  __syncthreads();
  if (lane != 0 || !in) return;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[k] = 0.0;
    for (int i = 0; i < 8; ++i) v[k] += red[k][i][cl];
  }
  auto put = [&](float* p, double x) { if (p) p[col] = (float)((d.accumulate ? (double)p[col] : 0.0) + x); };
  if (d.dh) { put(d.dw_pre, v[0]); put(d.db_pre, v[1]); }
  if (d.f) { put(d.dscale, w * v[2] + b * v[3]); put(d.dw_post, s * v[2]); put(d.db_post, s * v[3]); }
}

// ---------------------------------------------------------------------------------------------------------------- launches
// lanes, kind of team and channels per lane for rows of C channels (res_norm.hip)
void res_norm_team(int C, int* T, int* wave, int* nv);
template <int XT, int FT, int NV, bool WAVE, bool EACH, bool BIAS, bool NARROW = false>
static void fwd_go(const mscl_res_norm_desc& d, int T, unsigned grid, int64_t share, hipStream_t st) {
  const FastDiv g = make_fastdiv(d.gate && d.rows_per_gate < d.rows ? (int)d.rows_per_gate : 1);        // below 2^30, as it has to be
  hipLaunchKernelGGL((res_norm_fwd_kernel<XT, FT, NV, WAVE, EACH, BIAS, NARROW>), dim3(grid), dim3(WAVE ? 256 : T), 0, st, d, T, g, share);
}
template <int XT, int FT, int NV, bool WAVE>
static void fwd_launch(const mscl_res_norm_desc& d, int T, unsigned grid, int64_t share, hipStream_t st) {
  const bool each = d.gate && d.rows_per_gate == 1, bias = d.b_post || d.b_pre;
  if constexpr (WAVE) {
    if (d.C < 8) {
      if (each) fwd_go<XT, FT, NV, WAVE, true, true, true>(d, T, grid, share, st);
      else fwd_go<XT, FT, NV, WAVE, false, true, true>(d, T, grid, share, st);
      return;
    }
  }
  if (each) { if (bias) fwd_go<XT, FT, NV, WAVE, true, true>(d, T, grid, share, st); else fwd_go<XT, FT, NV, WAVE, true, false>(d, T, grid, share, st); }
  else { if (bias) fwd_go<XT, FT, NV, WAVE, false, true>(d, T, grid, share, st); else fwd_go<XT, FT, NV, WAVE, false, false>(d, T, grid, share, st); }
}
template <int XT, int FT>
void res_norm_fwd_types(const mscl_res_norm_desc& d, hipStream_t st) {
  int T, wave, nv;
  res_norm_team(d.C, &T, &wave, &nv);
  const int per = wave ? 256 / T : 1;
  // Each block takes its rows in one stretch, s to a team: short, so that the last blocks end together (32768 x 2048, fp32 / bf16: 172 us with
  // 16 rows a team, 161 with 8, 155 with 4, 158 with 2), or so long that all blocks are resident at once.  Of these the s is taken with the
  // fewest row times: rounds of the resident blocks (part of one more where they overlap) times s and one for a block's start.  (Against blocks
  // for 32 waves a CU at up to 4 rows: 1556 x 6040 fp32 / bf16, biases, 31 -> 22 us; 6696 x 3584 bf16 41 -> 36; 400 x 5000 12 -> 9.)
  const int waves = nv == 1 && !(d.b_post || d.b_pre) ? 5 : 4;             // a SIMD, by registers
  const int64_t resident = 256 * (wave ? waves : waves * 4 / (T / 64));
  int64_t share = per;
  double best = 1e30;
  for (int s = 1; s <= (wave ? 8 : 16); ++s) {
    const double n = (double)cdiv64(d.rows, s * per) / resident, whole = n <= 1.0 ? 1.0 : n + 0.5 < ceil(n) ? n + 0.5 : ceil(n);
    if ((s <= 4 || n <= 1.0) && whole * (s + 1) < best) { best = whole * (s + 1); share = s * per; }
  }
  const int64_t grid = cdiv64(d.rows, share);
  if (wave) fwd_launch<XT, FT, 1, true>(d, T, (unsigned)grid, share, st);
  else if (nv == 1) fwd_launch<XT, FT, 1, false>(d, T, (unsigned)grid, share, st);
  else fwd_launch<XT, FT, 2, false>(d, T, (unsigned)grid, share, st);
}
template <int XT, int FT, int NV, bool WAVE, int THREADS, int MODE, bool BIAS, bool NARROW = false>
static int bwd_go(const mscl_res_norm_desc& d, const BwdPlan& p, hipStream_t st) {
  constexpr int IN_LDS = bwd_in_lds(NV, THREADS, XT, MODE, BIAS);
  const int bytes = WAVE ? 256 * 8 * NV * 4 : IN_LDS / (BIAS ? 1 : 2) * NV * 32 * p.T;
  if constexpr (IN_LDS) {
    static std::atomic<uint64_t> told{0};             // a bit for each of the first 64 devices
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return (int)e;
    const uint64_t bit = dev < 64 ? (uint64_t)1 << dev : 0;
    if (!(told.load(std::memory_order_relaxed) & bit)) {
      e = hipFuncSetAttribute(reinterpret_cast<const void*>(res_norm_bwd_kernel<XT, FT, NV, WAVE, THREADS, MODE, BIAS, NARROW>), hipFuncAttributeMaxDynamicSharedMemorySize, 144 * 1024);
      if (e != hipSuccess) return (int)e;
      told.fetch_or(bit, std::memory_order_relaxed);
    }
  }
  hipLaunchKernelGGL((res_norm_bwd_kernel<XT, FT, NV, WAVE, THREADS, MODE, BIAS, NARROW>), dim3(p.blocks), dim3(WAVE ? 256 : p.T), bytes, st, d, p);
  MSCL_LAUNCH_CHECK();
  return 0;
}
template <int XT, int FT, int NV, bool WAVE, int THREADS>
static int bwd_launch(const mscl_res_norm_desc& d, const BwdPlan& p, hipStream_t st) {
  // the rare forms (rows below 8 channels, short runs per gate) carry the bias sums always
  if constexpr (WAVE) {
    if (d.C < 8) {
      if (p.mode == WHOLE) return bwd_go<XT, FT, NV, WAVE, THREADS, WHOLE, true, true>(d, p, st);
      if (p.mode == SPLIT) return bwd_go<XT, FT, NV, WAVE, THREADS, SPLIT, true, true>(d, p, st);
      return bwd_go<XT, FT, NV, WAVE, THREADS, EACH1, true, true>(d, p, st);
    }
  }
  if (p.mode == WHOLE) return bwd_go<XT, FT, NV, WAVE, THREADS, WHOLE, true>(d, p, st);
  if (d.b_post || d.b_pre) {
    if (p.mode == SPLIT) return bwd_go<XT, FT, NV, WAVE, THREADS, SPLIT, true>(d, p, st);
    return bwd_go<XT, FT, NV, WAVE, THREADS, EACH1, true>(d, p, st);
  }
  if (p.mode == SPLIT) return bwd_go<XT, FT, NV, WAVE, THREADS, SPLIT, false>(d, p, st);
  return bwd_go<XT, FT, NV, WAVE, THREADS, EACH1, false>(d, p, st);
}
template <int XT, int FT>
int res_norm_bwd_types(const mscl_res_norm_desc& d, const BwdPlan& p, hipStream_t st) {
  const int rc = p.wave ? bwd_launch<XT, FT, 1, true, 256>(d, p, st)
               : p.nv == 2 ? bwd_launch<XT, FT, 2, false, 1024>(d, p, st)
               : p.T <= 512 ? bwd_launch<XT, FT, 1, false, 512>(d, p, st)
               : p.T <= 768 ? bwd_launch<XT, FT, 1, false, 768>(d, p, st)        // 168 registers a lane; 1024 lanes leave 128
               : bwd_launch<XT, FT, 1, false, 1024>(d, p, st);
  if (rc) return rc;
  // few columns a block for narrow rows (few blocks), whole 64-byte segments for wide ones (C = 64 / 1024, 3 M elements, a training pass: 36 / 49 us
  // with 4 columns, 38 / 38 with 16; this launch at C = 1000 / 768 / 568: 29 / 18 / 19 us with 4, 17 / 13 / 13 with 8, 18 / 13 / 17 with 16)
  const int cols = d.C < 512 ? 4 : d.C < 1024 ? 8 : 16;
  int lanes = 1;
  if (d.gate && p.mode == SPLIT) while (lanes * 2 * p.gates <= 512 / cols && lanes * 2 <= p.per_gate) lanes *= 2;
  const dim3 grid((d.C + cols - 1) / cols);
  if (cols == 4) hipLaunchKernelGGL((res_norm_finish_kernel<FT, 4>), grid, dim3(512), 0, st, d, p, lanes);
  else if (cols == 8) hipLaunchKernelGGL((res_norm_finish_kernel<FT, 8>), grid, dim3(512), 0, st, d, p, lanes);
  else hipLaunchKernelGGL((res_norm_finish_kernel<FT, 16>), grid, dim3(512), 0, st, d, p, lanes);
  MSCL_LAUNCH_CHECK();
  return 0;
}
