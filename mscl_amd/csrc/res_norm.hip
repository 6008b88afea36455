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
// A TEAM of lanes owns a row: 1 .. 16 or 64 lanes of a wave (C <= 1024; sums by DPP), or the whole block (sums through LDS).  A lane
// holds NV x 8 channels in registers, so a row is read once.  VEC: 16-byte accesses, a lane's 8 channels adjacent; otherwise element
// accesses with a team's lanes on adjacent channels (odd C, odd strides, unaligned pointers).
#include "common.h"
#include <hip/hip_fp16.h>

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
template <int T> __device__ __forceinline__ void ld8(const void* p, int64_t e, float* v) {
  if (T == MSCL_F32) {
    *(float4*)v = *(const float4*)((const float*)p + e);
    *(float4*)(v + 4) = *(const float4*)((const float*)p + e + 4);
  } else {
    const uint4 u = *(const uint4*)((const uint16_t*)p + e);
    if (T == MSCL_BF16) unpack8(u, v);
    else {
      const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) { v[2 * i] = h2f((uint16_t)w[i]); v[2 * i + 1] = h2f((uint16_t)(w[i] >> 16)); }
    }
  }
}
template <int T> __device__ __forceinline__ void st8(void* p, int64_t e, const float* v) {
  if (T == MSCL_F32) {
    *(float4*)((float*)p + e) = *(const float4*)v;
    *(float4*)((float*)p + e + 4) = *(const float4*)(v + 4);
  } else if (T == MSCL_BF16) {
    *(uint4*)((uint16_t*)p + e) = pack8(v);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)f2h(v[2 * i]) | (uint32_t)f2h(v[2 * i + 1]) << 16;
    *(uint4*)((uint16_t*)p + e) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// a lane's channels of a row: value (q, i) is channel VEC ? (q T + lane) 8 + i : (q 8 + i) T + lane
template <int NV, bool VEC> struct Cols {
  int lane, T, C;
  __device__ __forceinline__ int col(int q, int i) const { return VEC ? (q * T + lane) * 8 + i : (q * 8 + i) * T + lane; }
  __device__ __forceinline__ bool has(int q, int i) const { return col(q, VEC ? 0 : i) < C; }
  template <int TY> __device__ __forceinline__ void load(const void* p, int64_t row, float (&v)[NV][8], float fill = 0.f) const {
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      if (VEC) {
        if (has(q, 0)) ld8<TY>(p, row + col(q, 0), v[q]);
        else
#pragma unroll
          for (int i = 0; i < 8; ++i) v[q][i] = fill;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[q][i] = has(q, i) ? ld1<TY>(p, row + col(q, i)) : fill;
      }
    }
  }
  // a per-channel vector; a missing one is all `one`
  __device__ __forceinline__ void load_vec(const float* p, float one, float (&v)[NV][8]) const {
    if (p) load<MSCL_F32>(p, 0, v, 0.f);
    else
#pragma unroll
      for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[q][i] = one;
  }
  template <int TY> __device__ __forceinline__ void store(void* p, int64_t row, const float (&v)[NV][8]) const {
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      if (VEC) { if (has(q, 0)) st8<TY>(p, row + col(q, 0), v[q]); }
      else
#pragma unroll
        for (int i = 0; i < 8; ++i) if (has(q, i)) st1<TY>(p, row + col(q, i), v[q][i]);
    }
  }
};

// team sums.  WAVE: T in {1, 2, 4, 8, 16, 64}.  Block teams: waves meet in LDS; two alternating slots make one barrier per sum enough
// (a slot is written again only by waves that have passed the barrier of the sum between, i.e. after every wave has read it).
template <int CTRL> __device__ __forceinline__ float dpp_add(float v) {
  return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
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
    return v;
  }
  __device__ __forceinline__ float2 sum2(float a, float b, bool want_b) {
    if (WAVE) return make_float2(wsum(a), want_b ? wsum(b) : 0.f);
    a = wave_sum(a);
    if (want_b) b = wave_sum(b);
    const int w = threadIdx.x >> 6, nw = blockDim.x >> 6;
    float2* s = red + slot * 16;
    slot ^= 1;
    if ((threadIdx.x & 63) == 0) s[w] = make_float2(a, b);
    __syncthreads();
    float2 t = s[0];
    for (int i = 1; i < nw; ++i) { const float2 u = s[i]; t.x += u.x; t.y += u.y; }
    return t;
  }
  __device__ __forceinline__ float sum(float a) { return sum2(a, 0.f, false).x; }
};

__device__ __forceinline__ float act_fwd(int act, float g) {
  if (act == MSCL_GATE_SIGMOID) return 1.f / (1.f + expf(-g));
  if (act == MSCL_GATE_TANH) return tanhf(g);
  return g;
}
// a'(g) = e / (1 + e)^2 with e = exp(-|g|) (sigmoid), 4 e / (1 + e)^2 with e = exp(-2 |g|) (tanh): no difference of near numbers, which
// a (1 - a) and 1 - a^2 are for a saturated gate
__device__ __forceinline__ float act_slope(int act, float g) {
  if (act == MSCL_GATE_LINEAR) return 1.f;
  const bool th = act == MSCL_GATE_TANH;
  const float e = expf(-fabsf(g) * (th ? 2.f : 1.f)), q = 1.f / (1.f + e);
  return (th ? 4.f : 1.f) * e * q * q;
}

// mean and 1 / deviation of a row held in v (kind 1: mean 0); the second moment is taken about the mean, in a second register pass
template <int NV, bool VEC, bool WAVE>
__device__ __forceinline__ float2 row_stats(const float (&v)[NV][8], int kind, float inv_c, float eps, const Cols<NV, VEC>& c, Team<WAVE>& team) {
  float mu = 0.f;
  if (kind == MSCL_NORM_LAYER) {
    float s = 0.f;
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
      for (int i = 0; i < 8; ++i) s += v[q][i];              // channels past C are zero
    mu = team.sum(s) * inv_c;
  }
  float s = 0.f;
#pragma unroll
  for (int q = 0; q < NV; ++q)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float d = c.has(q, i) ? v[q][i] - mu : 0.f;
      s += d * d;
    }
  const float var = team.sum(s) * inv_c;
  return make_float2(mu, 1.f / sqrtf(var + eps));
}
}  // namespace

template <int XT, int FT, int NV, bool VEC, bool WAVE>
__global__ __launch_bounds__(WAVE ? 256 : 1024) void res_norm_fwd_kernel(mscl_res_norm_desc d, int T, FastDiv gdiv) {
  __shared__ float2 red[32];
  Team<WAVE> team{T, red, 0};
  const int per = WAVE ? 256 / T : 1, sub = WAVE ? (int)threadIdx.x / T : 0;
  const Cols<NV, VEC> c{WAVE ? (int)threadIdx.x % T : (int)threadIdx.x, T, d.C};
  const float inv_c = 1.f / (float)d.C;
  for (int64_t r = (int64_t)blockIdx.x * per + sub; r < d.rows; r += (int64_t)gridDim.x * per) {
    float x[NV][8];
    c.template load<XT>(d.x, r * d.ld_x, x);
    if (d.f) {
      float f[NV][8], w[NV][8];
      c.template load<FT>(d.f, r * d.ld_f, f);
      if (d.post) {
        const float2 st = row_stats<NV, VEC, WAVE>(f, d.post, inv_c, d.eps, c, team);
        if (c.lane == 0) {
          if (d.mean_f) d.mean_f[r] = st.x;
          if (d.rstd_f) d.rstd_f[r] = st.y;
        }
#pragma unroll
        for (int q = 0; q < NV; ++q)
#pragma unroll
          for (int i = 0; i < 8; ++i) f[q][i] = (f[q][i] - st.x) * st.y;
      }
      if (d.w_post) {
        c.load_vec(d.w_post, 1.f, w);
#pragma unroll
        for (int q = 0; q < NV; ++q)
#pragma unroll
          for (int i = 0; i < 8; ++i) f[q][i] *= w[q][i];
      }
      if (d.b_post) {
        c.load_vec(d.b_post, 0.f, w);
#pragma unroll
        for (int q = 0; q < NV; ++q)
#pragma unroll
          for (int i = 0; i < 8; ++i) f[q][i] += w[q][i];
      }
      if (d.scale) {
        c.load_vec(d.scale, 1.f, w);
#pragma unroll
        for (int q = 0; q < NV; ++q)
#pragma unroll
          for (int i = 0; i < 8; ++i) f[q][i] *= w[q][i];
      }
      if (d.gate) {
        c.template load<FT>(d.gate, (int64_t)fdiv((int)r, gdiv) * d.C, w);
#pragma unroll
        for (int q = 0; q < NV; ++q)
#pragma unroll
          for (int i = 0; i < 8; ++i) f[q][i] *= act_fwd(d.gate_act, w[q][i]);
      }
#pragma unroll
      for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[q][i] = c.has(q, i) ? x[q][i] + f[q][i] : 0.f;
      c.template store<XT>(d.y, r * d.C, x);
    }
    if (d.pre) {
      float w[NV][8];
      const float2 st = row_stats<NV, VEC, WAVE>(x, d.pre, inv_c, d.eps, c, team);
      if (c.lane == 0) {
        if (d.mean_y) d.mean_y[r] = st.x;
        if (d.rstd_y) d.rstd_y[r] = st.y;
      }
      c.load_vec(d.w_pre, 1.f, w);
#pragma unroll
      for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[q][i] = (x[q][i] - st.x) * st.y * w[q][i];
      if (d.b_pre) {
        c.load_vec(d.b_pre, 0.f, w);
#pragma unroll
        for (int q = 0; q < NV; ++q)
#pragma unroll
          for (int i = 0; i < 8; ++i) x[q][i] += w[q][i];
      }
      c.template store<FT>(d.h, r * d.C, x);
    }
  }
}

// Which rows a block of the backward pass takes, and which column sums it leaves.
//   split  the gates are long runs of rows (or there is one, or none): `per_gate` blocks share the rows of a gate, their T1 / T2 stay
//          apart per gate until the second launch has added them up and applied a and a'
//   whole  the gates are short (down to one row): a team takes whole gates, applies a itself and writes dgate
struct BwdPlan { int T, wave, nv, vec, whole, per_gate, gates, blocks, rows_per_gate; };

template <int XT, int FT, int NV, bool VEC, bool WAVE, bool WHOLE>
__global__ __launch_bounds__(WAVE ? 256 : 1024) void res_norm_bwd_kernel(mscl_res_norm_desc d, BwdPlan pl) {
  extern __shared__ float lds[];                    // wave teams: [256][8 NV] for the column sums of a block
  __shared__ float2 red[32];
  const int T = pl.T;
  Team<WAVE> team{T, red, 0};
  const int per = WAVE ? 256 / T : 1, sub = WAVE ? (int)threadIdx.x / T : 0;
  const Cols<NV, VEC> c{WAVE ? (int)threadIdx.x % T : (int)threadIdx.x, T, d.C};
  const float inv_c = 1.f / (float)d.C;
  float sw[NV][8], sb[NV][8], w2[NV][8], a[NV][8], logit[WHOLE ? NV : 1][8];
  float U1[NV][8] = {}, U2[NV][8] = {}, T1[NV][8] = {}, T2[NV][8] = {}, t1[NV][8] = {}, t2[NV][8] = {};
  if (d.f) {
    float s[NV][8];
    c.load_vec(d.scale, 1.f, s);
    c.load_vec(d.w_post, 1.f, sw);
    c.load_vec(d.b_post, 0.f, sb);
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
      for (int i = 0; i < 8; ++i) { sw[q][i] *= s[q][i]; sb[q][i] *= s[q][i]; a[q][i] = 1.f; }
  }
  c.load_vec(d.w_pre, 1.f, w2);

  auto row = [&](int64_t r) {
    float x[NV][8], n[NV][8], t[NV][8];
    float rf = 1.f;
    c.template load<XT>(d.x, r * d.ld_x, x);
    if (d.f) c.template load<FT>(d.f, r * d.ld_f, n);
    if (d.dy) c.template load<XT>(d.dy, r * d.C, t);
    else
#pragma unroll
      for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int i = 0; i < 8; ++i) t[q][i] = 0.f;
    if (d.f) {
      if (d.post) {
        const float mu = d.post == MSCL_NORM_LAYER ? d.mean_f[r] : 0.f;
        rf = d.rstd_f[r];
#pragma unroll
        for (int q = 0; q < NV; ++q)
#pragma unroll
          for (int i = 0; i < 8; ++i) n[q][i] = c.has(q, i) ? (n[q][i] - mu) * rf : 0.f;
      }
#pragma unroll
      for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[q][i] += a[q][i] * (sw[q][i] * n[q][i] + sb[q][i]);        // y
    }
    if (d.dh) {
      float g[NV][8];
      c.template load<FT>(d.dh, r * d.C, g);
      const float mu = d.pre == MSCL_NORM_LAYER ? d.mean_y[r] : 0.f, ry = d.rstd_y[r];
      float c1 = 0.f, c0 = 0.f;
#pragma unroll
      for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float yh = c.has(q, i) ? (x[q][i] - mu) * ry : 0.f;
          x[q][i] = yh;
          U1[q][i] += g[q][i] * yh;
          U2[q][i] += g[q][i];
          g[q][i] *= w2[q][i];
          c1 += g[q][i] * yh;
          c0 += g[q][i];
        }
      const float2 s = team.sum2(c1, c0, d.pre == MSCL_NORM_LAYER);
      const float m1 = s.x * inv_c, m0 = d.pre == MSCL_NORM_LAYER ? s.y * inv_c : 0.f;
#pragma unroll
      for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int i = 0; i < 8; ++i) t[q][i] += ry * (g[q][i] - m0 - x[q][i] * m1);
    }
    if (d.dx) c.template store<XT>(d.dx, r * d.C, t);
    if (!d.f) return;
    float k1 = 0.f, k0 = 0.f;
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float ti = c.has(q, i) ? t[q][i] : 0.f;
        T1[q][i] += ti * n[q][i];
        T2[q][i] += ti;
        t[q][i] = ti * a[q][i] * sw[q][i];
        k1 += t[q][i] * n[q][i];
        k0 += t[q][i];
      }
    if (!d.df) return;
    if (d.post) {
      const float2 s = team.sum2(k1, k0, d.post == MSCL_NORM_LAYER);
      const float m1 = s.x * inv_c, m0 = d.post == MSCL_NORM_LAYER ? s.y * inv_c : 0.f;
#pragma unroll
      for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int i = 0; i < 8; ++i) t[q][i] = rf * (t[q][i] - m0 - n[q][i] * m1);
    }
    c.template store<FT>(d.df, r * d.C, t);
  };
  auto load_gate = [&](int64_t g) {
    c.template load<FT>(d.gate, g * d.C, a);
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (WHOLE) logit[q][i] = a[q][i];
        a[q][i] = act_fwd(d.gate_act, a[q][i]);
      }
  };

  if (WHOLE) {
    for (int64_t g = (int64_t)blockIdx.x * per + sub; g < pl.gates; g += (int64_t)gridDim.x * per) {
      load_gate(g);
      for (int64_t r = g * pl.rows_per_gate; r < (g + 1) * pl.rows_per_gate; ++r) row(r);
#pragma unroll
      for (int q = 0; q < NV; ++q)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          t1[q][i] += a[q][i] * T1[q][i];
          t2[q][i] += a[q][i] * T2[q][i];
          a[q][i] = act_slope(d.gate_act, logit[q][i]) * (sw[q][i] * T1[q][i] + sb[q][i] * T2[q][i]);
          T1[q][i] = T2[q][i] = 0.f;
        }
      if (d.dgate) c.template store<FT>(d.dgate, g * d.C, a);
    }
  } else {
    const int64_t g = blockIdx.x / pl.per_gate, j = blockIdx.x % pl.per_gate;
    const int64_t share = (pl.rows_per_gate + pl.per_gate - 1) / pl.per_gate, r0 = g * pl.rows_per_gate;
    const int64_t end = r0 + (share * (j + 1) < pl.rows_per_gate ? share * (j + 1) : pl.rows_per_gate);
    if (d.gate) load_gate(g);
    for (int64_t r = r0 + share * j + sub; r < end; r += per) row(r);
  }

  // the block's column sums: [4][C] floats (U1, U2, T1, T2; whole gates: t1, t2 in the place of T1, T2)
  float* out = d.ws + (int64_t)blockIdx.x * 4 * d.C;
  for (int k = 0; k < 4; ++k) {
    if ((k < 2 ? !d.dh : !d.f) || (k == 1 && !d.db_pre) || (k == 3 && !d.b_post)) continue;       // block-uniform
    float (&v)[NV][8] = k == 0 ? U1 : k == 1 ? U2 : k == 2 ? (WHOLE ? t1 : T1) : (WHOLE ? t2 : T2);
    if (!WAVE) { c.template store<MSCL_F32>(out + (int64_t)k * d.C, 0, v); continue; }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < NV; ++q)
#pragma unroll
      for (int i = 0; i < 8; ++i) lds[sub * T * 8 * NV + c.col(q, i)] = v[q][i];
    __syncthreads();
    for (int e = threadIdx.x; e < d.C; e += 256) {
      float s = 0.f;
      for (int u = 0; u < per; ++u) s += lds[u * T * 8 * NV + e];
      out[(int64_t)k * d.C + e] = s;
    }
  }
}

// Adds the blocks' column sums: 16 columns x 64 lanes per block.  Split gates: lanes_per_gate lanes share the blocks of a gate, the first
// of them writes dgate and goes on with a T1, a T2.
template <int FT>
__global__ __launch_bounds__(1024) void res_norm_finish_kernel(mscl_res_norm_desc d, BwdPlan pl, int lanes_per_gate) {
  __shared__ double red[2][64][16];
  const int cl = threadIdx.x & 15, lane = threadIdx.x >> 4;
  const int col = blockIdx.x * 16 + cl;
  const bool in = col < d.C;
  const int64_t stride = (int64_t)4 * d.C;
  auto total = [&](double v) {                       // over the 64 lanes of a column, in a fixed tree
    __syncthreads();
    red[0][lane][cl] = v;
    __syncthreads();
    for (int w = 32; w > 0; w >>= 1) {
      if (lane < w) red[0][lane][cl] += red[0][lane + w][cl];
      __syncthreads();
    }
    return red[0][0][cl];
  };
  auto plain = [&](int k) {
    double s = 0.0;
    if (in)
#pragma unroll 8
      for (int b = lane; b < pl.blocks; b += 64) s += (double)d.ws[b * stride + (int64_t)k * d.C + col];
    return total(s);
  };
  auto put = [&](float* p, double v) { if (p && in && lane == 0) p[col] = (float)((d.accumulate ? (double)p[col] : 0.0) + v); };
  if (d.dh) {
    if (d.dw_pre) put(d.dw_pre, plain(0));
    if (d.db_pre) put(d.db_pre, plain(1));
  }
  if (!d.f) return;
  const double w = in && d.w_post ? (double)d.w_post[col] : 1.0, b = in && d.b_post ? (double)d.b_post[col] : 0.0;
  const double s = in && d.scale ? (double)d.scale[col] : 1.0;
  double t1, t2 = 0.0;
  if (pl.whole || !d.gate) {
    t1 = plain(2);
    if (d.b_post) t2 = plain(3);
  } else {
    const int at_once = 64 / lanes_per_gate, mine = lane / lanes_per_gate, part = lane % lanes_per_gate;
    double a1 = 0.0, a2 = 0.0;
    for (int g0 = 0; g0 < pl.gates; g0 += at_once) {
      const int g = g0 + mine;
      double s1 = 0.0, s2 = 0.0;
      if (in && g < pl.gates)
#pragma unroll 4
        for (int j = part; j < pl.per_gate; j += lanes_per_gate) {
          const float* p = d.ws + ((int64_t)g * pl.per_gate + j) * stride + col;
          s1 += (double)p[2 * (int64_t)d.C];
          if (d.b_post) s2 += (double)p[3 * (int64_t)d.C];
        }
      if (lanes_per_gate > 1) {
        __syncthreads();
        red[0][lane][cl] = s1;
        red[1][lane][cl] = s2;
        __syncthreads();
        if (part == 0)
          for (int i = 1; i < lanes_per_gate; ++i) { s1 += red[0][lane + i][cl]; s2 += red[1][lane + i][cl]; }
      }
      if (part == 0 && in && g < pl.gates) {
        const float logit = ld1<FT>(d.gate, (int64_t)g * d.C + col), a = act_fwd(d.gate_act, logit);
        a1 += (double)a * s1;
        a2 += (double)a * s2;
        if (d.dgate) st1<FT>(d.dgate, (int64_t)g * d.C + col, (float)(s * (double)act_slope(d.gate_act, logit) * (w * s1 + b * s2)));
      }
    }
    t1 = total(a1);
    if (d.b_post) t2 = total(a2);
  }
  put(d.dscale, w * t1 + b * t2);
  put(d.dw_post, s * t1);
  put(d.db_post, s * t2);
}

// ---------------------------------------------------------------------------------------------------------------- host
static int res_norm_check(const mscl_res_norm_desc* d) {
  if (!d || !d->x || d->rows <= 0 || d->C <= 0 || !(d->eps > 0.f)) return MSCL_E_ARG;
  if (!d->f && !d->pre) return MSCL_E_ARG;
  if (d->rows > 0x7FFFFFFF || d->C > MSCL_RES_NORM_MAX_C) return MSCL_E_SHAPE;
  if (d->post < 0 || d->post > 2 || d->pre < 0 || d->pre > 2 || d->gate_act < 0 || d->gate_act > 2) return MSCL_E_ARG;
  const bool t16 = d->f_type == MSCL_BF16 || d->f_type == MSCL_F16;
  if (!(d->x_type == d->f_type && (t16 || d->f_type == MSCL_F32)) && !(d->x_type == MSCL_F32 && t16)) return MSCL_E_SHAPE;
  if (d->ld_x < d->C || (d->f && d->ld_f < d->C)) return MSCL_E_STRIDE;
  if (d->gate && (!d->f || d->rows_per_gate <= 0 || d->rows % d->rows_per_gate)) return MSCL_E_SHAPE;
  return 0;
}
static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
static bool res_norm_vec(const mscl_res_norm_desc* d) {
  const int xs = d->x_type == MSCL_F32 ? 4 : 2, fs = d->f_type == MSCL_F32 ? 4 : 2;
  const void* p[] = {d->x, d->f, d->gate, d->scale, d->w_post, d->b_post, d->w_pre, d->b_pre, d->y, d->h, d->dy, d->dh, d->dx, d->df, d->dgate, d->ws};
  for (const void* q : p) if (!aligned16(q)) return false;
  return d->C % 8 == 0 && d->ld_x * xs % 16 == 0 && (!d->f || d->ld_f * fs % 16 == 0);
}
// lanes of a row: the fewest that hold it at 8 NV channels each
static void res_norm_team(int C, int max_wave_nv, int* T, int* wave, int* nv) {
  *nv = 1;
  for (int t = 1; t <= 16; t *= 2) if (C <= 8 * t) { *T = t; *wave = 1; return; }
  if (C <= 512) { *T = 64; *wave = 1; if (max_wave_nv == 2 && C <= 256) { *T = 16; *nv = 2; } return; }
  if (C <= 1024 && max_wave_nv == 2) { *T = 64; *wave = 1; *nv = 2; return; }
  *wave = 0;
  *nv = C > 8192 ? 2 : 1;
  const int need = (C + 8 * *nv - 1) / (8 * *nv);
  *T = (need + 63) / 64 * 64;
}

template <int XT, int FT, int NV, bool VEC>
static void fwd_launch(const mscl_res_norm_desc& d, int T, int wave, unsigned grid, FastDiv g, hipStream_t st) {
  if (wave) hipLaunchKernelGGL((res_norm_fwd_kernel<XT, FT, NV, VEC, true>), dim3(grid), dim3(256), 0, st, d, T, g);
  else hipLaunchKernelGGL((res_norm_fwd_kernel<XT, FT, NV, VEC, false>), dim3(grid), dim3(T), 0, st, d, T, g);
}
template <int XT, int FT>
static void fwd_types(const mscl_res_norm_desc& d, hipStream_t st) {
  int T, wave, nv;
  res_norm_team(d.C, 2, &T, &wave, &nv);
  const int per = wave ? 256 / T : 1;
  int64_t grid = cdiv64(d.rows, per);
  if (grid > 65536) grid = 65536;
  const FastDiv g = make_fastdiv(d.gate ? (int)d.rows_per_gate : 1);
  const bool vec = res_norm_vec(&d);
  if (nv == 1) { if (vec) fwd_launch<XT, FT, 1, true>(d, T, wave, (unsigned)grid, g, st); else fwd_launch<XT, FT, 1, false>(d, T, wave, (unsigned)grid, g, st); }
  else { if (vec) fwd_launch<XT, FT, 2, true>(d, T, wave, (unsigned)grid, g, st); else fwd_launch<XT, FT, 2, false>(d, T, wave, (unsigned)grid, g, st); }
}
extern "C" int mscl_res_norm_fwd(const mscl_res_norm_desc* d, void* stream) {
  const int rc = res_norm_check(d);
  if (rc) return rc;
  if ((d->f && !d->y) || (d->pre && !d->h)) return MSCL_E_ARG;
  hipStream_t st = (hipStream_t)stream;
  if (d->x_type == MSCL_BF16) fwd_types<MSCL_BF16, MSCL_BF16>(*d, st);
  else if (d->x_type == MSCL_F16) fwd_types<MSCL_F16, MSCL_F16>(*d, st);
  else if (d->f_type == MSCL_F32) fwd_types<MSCL_F32, MSCL_F32>(*d, st);
  else if (d->f_type == MSCL_BF16) fwd_types<MSCL_F32, MSCL_BF16>(*d, st);
  else fwd_types<MSCL_F32, MSCL_F16>(*d, st);
  MSCL_LAUNCH_CHECK();
  return 0;
}

static BwdPlan bwd_plan(const mscl_res_norm_desc* d) {
  BwdPlan p;
  res_norm_team(d->C, 1, &p.T, &p.wave, &p.nv);
  p.vec = res_norm_vec(d);
  const int per = p.wave ? 256 / p.T : 1;
  // enough blocks to fill 256 CUs with 16 waves each; every block costs 4 C floats of column sums
  int target = p.wave ? 1024 : 4096 / (p.T / 64);
  if (target > 2048) target = 2048;
  p.rows_per_gate = (int)(d->gate ? d->rows_per_gate : d->rows);
  p.gates = (int)(d->rows / p.rows_per_gate);
  p.whole = d->gate && (p.rows_per_gate < 16 || p.gates >= 4 * target * per);
  if (p.whole) {
    p.per_gate = 1;
    const int64_t need = cdiv64(p.gates, per);
    p.blocks = (int)(need < target ? need : target);
  } else {
    int pg = (target + p.gates - 1) / p.gates;
    const int64_t most = cdiv64(p.rows_per_gate, per);
    if (pg > most) pg = (int)most;
    p.per_gate = pg < 1 ? 1 : pg;
    p.blocks = p.per_gate * p.gates;
  }
  return p;
}
extern "C" int64_t mscl_res_norm_ws(const mscl_res_norm_desc* d) {
  if (res_norm_check(d)) return 0;
  return (int64_t)bwd_plan(d).blocks * 4 * d->C;
}
template <int XT, int FT, int NV, bool VEC, bool WAVE>
static void bwd_launch(const mscl_res_norm_desc& d, const BwdPlan& p, hipStream_t st) {
  const size_t lds = WAVE ? (size_t)256 * 8 * NV * 4 : 0;
  const int threads = WAVE ? 256 : p.T;
  if (p.whole) hipLaunchKernelGGL((res_norm_bwd_kernel<XT, FT, NV, VEC, WAVE, true>), dim3(p.blocks), dim3(threads), lds, st, d, p);
  else hipLaunchKernelGGL((res_norm_bwd_kernel<XT, FT, NV, VEC, WAVE, false>), dim3(p.blocks), dim3(threads), lds, st, d, p);
}
template <int XT, int FT>
static int bwd_types(const mscl_res_norm_desc& d, const BwdPlan& p, hipStream_t st) {
  if (p.wave) { if (p.vec) bwd_launch<XT, FT, 1, true, true>(d, p, st); else bwd_launch<XT, FT, 1, false, true>(d, p, st); }
  else if (p.nv == 1) { if (p.vec) bwd_launch<XT, FT, 1, true, false>(d, p, st); else bwd_launch<XT, FT, 1, false, false>(d, p, st); }
  else { if (p.vec) bwd_launch<XT, FT, 2, true, false>(d, p, st); else bwd_launch<XT, FT, 2, false, false>(d, p, st); }
  MSCL_LAUNCH_CHECK();
  int lanes = 1;
  if (d.gate && !p.whole) while (lanes * 2 * p.gates <= 64 && lanes * 2 <= p.per_gate) lanes *= 2;
  hipLaunchKernelGGL(res_norm_finish_kernel<FT>, dim3((d.C + 15) / 16), dim3(1024), 0, st, d, p, lanes);
  MSCL_LAUNCH_CHECK();
  return 0;
}
extern "C" int mscl_res_norm_bwd(const mscl_res_norm_desc* d, void* stream) {
  const int rc = res_norm_check(d);
  if (rc) return rc;
  if (!d->dy && !d->dh) return MSCL_E_ARG;
  if ((d->dh && (!d->pre || !d->rstd_y || (d->pre == MSCL_NORM_LAYER && !d->mean_y)))) return MSCL_E_ARG;
  if (d->f && d->post && (!d->rstd_f || (d->post == MSCL_NORM_LAYER && !d->mean_f))) return MSCL_E_ARG;
  const BwdPlan p = bwd_plan(d);
  if (!d->ws || d->ws_floats < (int64_t)p.blocks * 4 * d->C) return MSCL_E_ARG;
  hipStream_t st = (hipStream_t)stream;
  if (d->x_type == MSCL_BF16) return bwd_types<MSCL_BF16, MSCL_BF16>(*d, p, st);
  if (d->x_type == MSCL_F16) return bwd_types<MSCL_F16, MSCL_F16>(*d, p, st);
  if (d->f_type == MSCL_F32) return bwd_types<MSCL_F32, MSCL_F32>(*d, p, st);
  if (d->f_type == MSCL_BF16) return bwd_types<MSCL_F32, MSCL_BF16>(*d, p, st);
  return bwd_types<MSCL_F32, MSCL_F16>(*d, p, st);
}
