// AdamW over many tensors in two or three launches, moments in 32 or in 8 bits (gfx950, HBM-bound).
//
// Mathematics (t counts steps, c = min(1, max_norm / (|g| + 1e-6)) with |g| the 2-norm over ALL tensors, g' = c g):
//   m = b1 m + (1 - b1) g'      v = b2 v + (1 - b2) g'^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// Launch 1 (adamw_prelude_kernel) advances the step counter on the device, so that a captured graph replays right, and finds c.  Launch 2
// (adamw_kernel) updates everything.  All sums are in a fixed order: replicas of a data-parallel job stay identical.
//
// 8-bit moments.  A block is 256 consecutive elements of one tensor = one wave x 4 elements, so its maximum is a DPP reduction and never
// leaves the wave.  It has an exponent byte for each moment (2^E, E from the largest magnitude); m is sign + 4 exponent + 3 mantissa bits
// below 2^E, v is 5 exponent + 3 mantissa bits: v ~ m^2 needs twice the range in octaves.  Powers of two make a code a slice of the fp32
// pattern: after ldexp has put the code's smallest normal exponent onto fp32's own, code = (bits + random) >> 20, subnormals included.
// The rounding is stochastic because b2 = 0.999 moves v by 0.1 % a step and 3 mantissa bits are 6-12 %: a nearest rounding would never move
// it.  p is updated from the moments BEFORE they are rounded.
//
// What bounds it (MI355X, where a copy of 4 GB runs at 4.8 TB/s and an in-place add at 5.9): memory.  Counters give the bytes of the
// formula and no more: 26 per element for 16-bit gradients and no shadow, 320 M elements in 1.48 ms = 5.6 TB/s; 33 M elements with fp32
// gradients, a clip and a shadow (30 bytes, 4 more where the gradient is read a second time, partly from the last-level cache): 25 us for the
// norm, 5 for the coefficient, 150 for the update.  8 bits: 16 bytes per element, 300 M in 0.85 ms = 5.7 TB/s with the vector units busy
// about four fifths of the time (80 instructions per element, two of them quarter-rate multiplies of the hash).
#include "common.h"
#include <hip/hip_fp16.h>
#include <cfloat>
#include <cstddef>

namespace {
constexpr int CHUNK = MSCL_ADAMW_CHUNK;        // elements a block of 256 threads takes: 4 vectors of 4 per thread and array, 16 loads in flight (32 bits)
constexpr int PARTS = MSCL_ADAMW_PARTS;
static_assert(CHUNK == 256 * 4 * 4 && MSCL_ADAMW_BLOCK == 64 * 4, "the kernels' shape");

struct Words { int64_t step; float c1, c2; uint32_t key, seed; float coef; uint32_t pad; };      // = the words buffer
static_assert(sizeof(Words) == MSCL_ADAMW_WORDS && offsetof(Words, seed) == 20, "the words buffer");

// The update passes once over far more memory than any cache holds: its accesses are marked non-temporal, which leaves the caches to the
// gradient between the launches (33 M elements, fp32 / clip / shadow: a step of 238 -> 200 us; 320 M without clip: 1611 -> 1507 us).
// Vectors of 4 elements are accessed at the alignment of one (the memory path of gfx950 takes any): a view that starts anywhere takes the same
// code, and of a tensor's last chunk only the vector that its end cuts goes element by element (161 tensors, 31.6 M elements: norm 34 -> 24 us).
typedef f32x4_t f32x4_at4 __attribute__((aligned(4)));
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2_t;
typedef u32x2_t u32x2_at2 __attribute__((aligned(2)));
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4_t;
__device__ __forceinline__ float4 ldnt(const float* p) {
  const f32x4_t v = __builtin_nontemporal_load((const f32x4_at4*)p);
  return make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void stnt(float* p, const float* v) {
  const f32x4_t u = {v[0], v[1], v[2], v[3]};
  __builtin_nontemporal_store(u, (f32x4_at4*)p);
}
__device__ __forceinline__ uint2 ldnt(const uint16_t* p) { const u32x2_t v = __builtin_nontemporal_load((const u32x2_at2*)p); return make_uint2(v[0], v[1]); }
__device__ __forceinline__ void stnt(uint16_t* p, uint2 v) { const u32x2_t u = {v.x, v.y}; __builtin_nontemporal_store(u, (u32x2_at2*)p); }
__device__ __forceinline__ uint2 ldnt(const uint2* p) { const u32x2_t v = __builtin_nontemporal_load((const u32x2_t*)p); return make_uint2(v[0], v[1]); }
__device__ __forceinline__ void stnt(uint4* p, uint4 v) { const u32x4_t u = {v.x, v.y, v.z, v.w}; __builtin_nontemporal_store(u, (u32x4_t*)p); }

__device__ __forceinline__ uint32_t mix32(uint32_t x) {          // finaliser of MurmurHash3 (Appleby, public domain)
  x ^= x >> 16; x *= 0x85EBCA6Bu; x ^= x >> 13; x *= 0xC2B2AE35u; x ^= x >> 16;
  return x;
}
template <int CTRL> __device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
  const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false);
  return v > o ? v : o;
}
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {      // largest of a wave's 64 values, wave-uniform
  v = dpp_max<0xB1>(v); v = dpp_max<0x4E>(v); v = dpp_max<0x124>(v); v = dpp_max<0x128>(v);
  const uint32_t a = (uint32_t)__builtin_amdgcn_readlane((int)v, 0), b = (uint32_t)__builtin_amdgcn_readlane((int)v, 16);
  const uint32_t c = (uint32_t)__builtin_amdgcn_readlane((int)v, 32), d = (uint32_t)__builtin_amdgcn_readlane((int)v, 48);
  const uint32_t e = a > b ? a : b, f = c > d ? c : d;
  return e > f ? e : f;
}
__device__ __forceinline__ double wave_dsum(double v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
  return v;
}

__device__ __forceinline__ float half2f(uint16_t h) { return __half2float(__ushort_as_half(h)); }
template <int GT> __device__ __forceinline__ float grad1(const void* g, int64_t e) {
  if (GT == MSCL_F32) return ((const float*)g)[e];
  const uint16_t h = ((const uint16_t*)g)[e];
  return GT == MSCL_BF16 ? bf2f(h) : half2f(h);
}
// 4 gradients from element e on; NT: for the last time
template <int GT, bool NT> __device__ __forceinline__ float4 grad4(const void* g, int64_t e) {
  if (GT == MSCL_F32) {
    if (NT) return ldnt((const float*)g + e);
    const f32x4_t v = *(const f32x4_at4*)((const float*)g + e);
    return make_float4(v[0], v[1], v[2], v[3]);
  }
  uint2 v;
  if (NT) v = ldnt((const uint16_t*)g + e);
  else { const u32x2_t u = *(const u32x2_at2*)((const uint16_t*)g + e); v = make_uint2(u[0], u[1]); }
  if (GT == MSCL_BF16)
    return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xFFFF0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xFFFF0000u));
  return make_float4(half2f((uint16_t)v.x), half2f((uint16_t)(v.x >> 16)), half2f((uint16_t)v.y), half2f((uint16_t)(v.y >> 16)));
}
// the same where the tensor ends at element n: zeros from there on
template <int GT, bool NT> __device__ __forceinline__ float4 grad4_end(const void* g, int64_t e, int64_t n) {
  if (e + 4 <= n) return grad4<GT, NT>(g, e);
  return make_float4(e < n ? grad1<GT>(g, e) : 0.f, e + 1 < n ? grad1<GT>(g, e + 1) : 0.f, e + 2 < n ? grad1<GT>(g, e + 2) : 0.f, 0.f);
}
__device__ __forceinline__ uint16_t f2half(float f) { return __half_as_ushort(__float2half_rn(f)); }
template <int ST> __device__ __forceinline__ uint16_t shadow1(float f) { return ST == MSCL_BF16 ? f2bf(f) : f2half(f); }

// codes <-> values; E: exponent field (biased by 127) of the block
__device__ __forceinline__ float decode_m(uint32_t c, int E) {
  const float a = ldexpf(__uint_as_float((c & 127u) << 20), 112 + E - 127);
  return __uint_as_float(__float_as_uint(a) | ((c & 128u) << 24));
}
__device__ __forceinline__ float decode_v(uint32_t c, int E) { return ldexpf(__uint_as_float(c << 20), 96 + E - 127); }
__device__ __forceinline__ uint32_t encode_m(float m, int E, uint32_t r16) {
  const uint32_t b = (__float_as_uint(ldexpf(fabsf(m), -112 - (E - 127))) + (r16 << 4)) >> 20;
  return (b < 127u ? b : 127u) | ((__float_as_uint(m) >> 24) & 128u);
}
__device__ __forceinline__ uint32_t encode_v(float v, int E, uint32_t r16) {
  uint32_t b = (__float_as_uint(ldexpf(v, -96 - (E - 127))) + (r16 << 4)) >> 20;
  b = b < 255u ? b : 255u;
  return (v > 0.f && b == 0u) ? 1u : b;          // a positive v stays positive: m / sqrt(v) must not become m / eps
}
// exponent field of a block from the largest magnitude's bits, after that magnitude is rounded up to 4 significant bits; 255 marks a
// block that holds an infinity or a NaN (it reads back as NaN)
__device__ __forceinline__ int block_exponent(uint32_t top) {
  if (top >= 0x7F800000u) return 255;
  const int e = (int)((top + 0x0FFFFFu) >> 23);
  return e < 1 ? 1 : e > 254 ? 254 : e;
}
}  // namespace

// min(1, max_norm / (norm + 1e-6)) from a block's sums of squares, one value per wave in red; a NaN norm stays a NaN
__device__ __forceinline__ float clip_coef(const mscl_adamw_desc& d, const double* red, bool keep_norm) {
  const double norm = sqrt((red[0] + red[1]) + (red[2] + red[3])), c = d.max_norm / (norm + 1e-6);
  if (keep_norm) *d.grad_norm = (float)norm;
  return c > 1.0 ? 1.f : (float)c;
}

// Step counter, bias corrections and rounding key (block 0) and, with a clip, a partial sum of squares per block in 64 bits.  The gradient
// is read a second time by the update: a clip by the global norm cannot know its coefficient before the last element.  What a block
// needs to know of its next chunk is fetched while this chunk's elements are on their way.
template <int GT>
__global__ __launch_bounds__(256) void adamw_prelude_kernel(mscl_adamw_desc d) {
  __shared__ double red[4];
  const int tid = threadIdx.x;
  Words* w = (Words*)d.words;
  if (blockIdx.x == 0 && tid == 0) {
    const int64_t t = w->step + 1;
    w->step = t;
    w->c1 = (float)(1.0 / (1.0 - pow(d.beta1, (double)t)));
    w->c2 = (float)(1.0 / sqrt(1.0 - pow(d.beta2, (double)t)));
    w->key = mix32((uint32_t)((uint64_t)w->seed + 0x9E3779B9ull * (uint64_t)t));
    if (d.max_norm <= 0.0) w->coef = 1.f;
  }
  if (d.max_norm <= 0.0) return;
  double s = 0.0;
  int chunk = blockIdx.x;                                    // the grid is no larger than the number of chunks
  int ti = d.chunk_tensor[chunk];
  int64_t n = d.tensors[ti].n, base = (int64_t)(chunk - d.tensors[ti].first_chunk) * CHUNK;
  const void* g = d.grads[ti];
  while (true) {
    const int64_t next = (int64_t)chunk + gridDim.x;
    const bool more = next < d.n_chunks;
    float4 v[4];
    if (base + CHUNK <= n) {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = grad4<GT, false>(g, base + k * 1024 + tid * 4);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = grad4_end<GT, false>(g, base + k * 1024 + tid * 4, n);
    }
    const int tn = more ? d.chunk_tensor[next] : ti;
    const int64_t n2 = d.tensors[tn].n, base2 = (next - d.tensors[tn].first_chunk) * CHUNK;
    const void* g2 = d.grads[tn];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      s += (double)v[k].x * v[k].x; s += (double)v[k].y * v[k].y; s += (double)v[k].z * v[k].z; s += (double)v[k].w * v[k].w;
    }
    if (!more) break;
    chunk = (int)next; ti = tn; n = n2; base = base2; g = g2;
  }
  s = wave_dsum(s);
  if ((tid & 63) == 0) red[tid >> 6] = s;
  __syncthreads();
  if (tid == 0) d.partials[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}
// the block's share of the partials, one sum per wave
__device__ __forceinline__ void add_partials(const mscl_adamw_desc& d, int parts, double* red) {
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += 256) s += d.partials[i];
  s = wave_dsum(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
}
__global__ __launch_bounds__(256) void adamw_coef_kernel(mscl_adamw_desc d, int parts) {
  __shared__ double red[4];
  add_partials(d, parts, red);
  if (threadIdx.x == 0) ((Words*)d.words)->coef = clip_coef(d, red, true);
}

// sqrt of four second moments by the 1-ulp instruction, which takes a subnormal for 0: where a wave has one (gradients below 1e-18, where a
// small eps is all that is left in the denominator), those go through it 2^64 times as large.  One class test an element otherwise.
__device__ __forceinline__ void sqrt4(const float* v, float* r) {
  bool sub = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[i] = __builtin_amdgcn_sqrtf(v[i]);
    sub |= __builtin_amdgcn_classf(v[i], 0x080);                  // positive subnormal
  }
  if (__builtin_amdgcn_ballot_w64(sub)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool low = v[i] < FLT_MIN;
      const float s = __builtin_amdgcn_sqrtf(low ? v[i] * 0x1p64f : v[i]);
      r[i] = low ? s * 0x1p-32f : s;
    }
  }
}

// A block owns CHUNK elements of one tensor; the loads of all four vectors of a thread go out before the first is used.
template <int GT, int ST, int BITS>
__global__ __launch_bounds__(256) void adamw_kernel(mscl_adamw_desc d, int parts) {
#pragma clang fp contract(off)
  __shared__ double red[4];
  const int tid = threadIdx.x;
  const int ti = d.chunk_tensor[blockIdx.x];
  const mscl_adamw_tensor* T = d.tensors + ti;
  float* __restrict__ p = T->p;
  const void* __restrict__ g = d.grads[ti];
  uint16_t* __restrict__ sh = T->shadow;
  const int64_t n = T->n, base = (int64_t)((int)blockIdx.x - T->first_chunk) * CHUNK, off = T->off + base;
  const Words* w = (const Words*)d.words;
  const bool whole = base + CHUNK <= n;

  float pv[4][4], gv[4][4];
  float4 mv[4], vv[4];
  uint32_t mc[4], vc[4];
  int em[4], ev[4];
  bool live[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int64_t e = base + k * 1024 + tid * 4;
    live[k] = base + k * 1024 + (tid & ~63) * 4 < n;            // wave-uniform: the 256 elements of this wave hold a live one
    if (whole) {
      *(float4*)pv[k] = ldnt(p + e);
      *(float4*)gv[k] = grad4<GT, true>(g, e);
    } else {
      if (e + 4 <= n) *(float4*)pv[k] = ldnt(p + e);
      else
#pragma unroll
        for (int i = 0; i < 4; ++i) pv[k][i] = e + i < n ? p[e + i] : 0.f;
      *(float4*)gv[k] = grad4_end<GT, true>(g, e, n);
    }
    if (live[k]) {                                               // the states are padded to whole 256-element blocks of zeros
      const int64_t s = off + k * 1024 + tid * 4;
      if (BITS == 32) {
        mv[k] = ldnt((const float*)d.m + s);
        vv[k] = ldnt((const float*)d.v + s);
      } else {
        mc[k] = __builtin_nontemporal_load((const uint32_t*)((const uint8_t*)d.m + s));
        vc[k] = __builtin_nontemporal_load((const uint32_t*)((const uint8_t*)d.v + s));
        em[k] = d.exponents[s >> 8];
        ev[k] = d.exponents[d.n_blocks + (s >> 8)];
      }
    }
  }
  float coef = w->coef;
  if (parts) {                                                   // not added up yet: every block does, in the same order
    add_partials(d, parts, red);
    coef = clip_coef(d, red, blockIdx.x == 0 && tid == 0);
  }
  const float lr = *d.lr * T->lr_mult;
  const float keep = 1.f - lr * T->decay, rate = lr * w->c1, c2 = w->c2, eps = (float)d.eps;
  const float b1 = (float)d.beta1, a1 = (float)(1.0 - d.beta1), b2 = (float)d.beta2, a2 = (float)(1.0 - d.beta2);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if (!live[k]) continue;
    const int64_t e = base + k * 1024 + tid * 4, s = off + k * 1024 + tid * 4;
    float m[4], v[4];
    if (BITS == 32) {
      *(float4*)m = mv[k]; *(float4*)v = vv[k];
    } else {
      const bool bad_m = em[k] == 255, bad_v = ev[k] == 255;     // a poisoned block reads back as NaN
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        m[i] = bad_m ? __builtin_nanf("") : decode_m(mc[k] >> (8 * i) & 255u, em[k]);
        v[i] = bad_v ? __builtin_nanf("") : decode_v(vc[k] >> (8 * i) & 255u, ev[k]);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // plain multiplies and adds, no fma: each rounding is that of the formula taken term by term, so that the 8-bit codes do not depend
      // on how a compiler contracts it.  sqrt and reciprocal are the 1-ulp instructions: 2^-22 of an update that is itself far below p.
      const float gi = gv[k][i] * coef;
      m[i] = m[i] * b1 + gi * a1;
      v[i] = v[i] * b2 + gi * gi * a2;
    }
    float root[4];
    sqrt4(v, root);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float den = root[i] * c2 + eps;
      pv[k][i] = pv[k][i] * keep - rate * m[i] * __builtin_amdgcn_rcpf(den);
    }
    if (whole || e + 4 <= n) {
      stnt(p + e, pv[k]);
      if (ST != MSCL_NONE) {
        uint2 b;
        b.x = shadow1<ST>(pv[k][0]) | (uint32_t)shadow1<ST>(pv[k][1]) << 16;
        b.y = shadow1<ST>(pv[k][2]) | (uint32_t)shadow1<ST>(pv[k][3]) << 16;
        stnt(sh + e, b);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (e + i < n) {
          p[e + i] = pv[k][i];
          if (ST != MSCL_NONE) sh[e + i] = shadow1<ST>(pv[k][i]);
        }
    }
    if (BITS == 32) {
      stnt((float*)d.m + s, m);
      stnt((float*)d.v + s, v);
    } else {
      uint32_t tm = 0, tv = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t a = __float_as_uint(m[i]) & 0x7FFFFFFFu, b = __float_as_uint(v[i]) & 0x7FFFFFFFu;
        tm = tm > a ? tm : a;
        tv = tv > b ? tv : b;
      }
      const int Em = block_exponent(wave_umax(tm)), Ev = block_exponent(wave_umax(tv));
      const uint32_t key = mix32((uint32_t)((uint64_t)s >> 32) + w->key);
      uint32_t cm = 0, cv = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t r = mix32(key ^ (uint32_t)(s + i));
        cm |= encode_m(m[i], Em, r & 0xFFFFu) << (8 * i);
        cv |= encode_v(v[i], Ev, r >> 16) << (8 * i);
      }
      __builtin_nontemporal_store(cm, (uint32_t*)((uint8_t*)d.m + s));
      __builtin_nontemporal_store(cv, (uint32_t*)((uint8_t*)d.v + s));
      if ((tid & 63) == 0) {
        d.exponents[s >> 8] = (uint8_t)Em;
        d.exponents[d.n_blocks + (s >> 8)] = (uint8_t)Ev;
      }
    }
  }
}

template <int GT, int ST>
static void adamw_update(const mscl_adamw_desc& d, int parts, hipStream_t st) {
  if (d.state_bits == 32) hipLaunchKernelGGL((adamw_kernel<GT, ST, 32>), dim3(d.n_chunks), dim3(256), 0, st, d, parts);
  else hipLaunchKernelGGL((adamw_kernel<GT, ST, 8>), dim3(d.n_chunks), dim3(256), 0, st, d, parts);
}
template <int GT>
static int adamw_launch(const mscl_adamw_desc& d, hipStream_t st) {
  int64_t blocks = 1;
  if (d.max_norm > 0.0) blocks = d.n_chunks < PARTS ? d.n_chunks : PARTS;
  hipLaunchKernelGGL(adamw_prelude_kernel<GT>, dim3((unsigned)blocks), dim3(256), 0, st, d);
  MSCL_LAUNCH_CHECK();
  // Up to 16 M elements the update's blocks add the partials up themselves, each all of them; from there on they are added once, in a launch of
  // its own: a step of 4 / 8 / 16 / 33 / 100 M elements 25 / 49 / 94 / 193 / 573 us without it, 30 / 53 / 93 / 179 / 546 us with it.  (The last
  // block of launch 1 adding them -- a ticket and a release per block -- took 90 us for 2048 blocks.)
  int parts = d.max_norm > 0.0 ? (int)blocks : 0;
  if (parts && d.n_chunks > 4096) {
    hipLaunchKernelGGL(adamw_coef_kernel, dim3(1), dim3(256), 0, st, d, parts);
    MSCL_LAUNCH_CHECK();
    parts = 0;
  }
  if (d.shadow_type == MSCL_NONE) adamw_update<GT, MSCL_NONE>(d, parts, st);
  else if (d.shadow_type == MSCL_BF16) adamw_update<GT, MSCL_BF16>(d, parts, st);
  else adamw_update<GT, MSCL_F16>(d, parts, st);
  MSCL_LAUNCH_CHECK();
  return 0;
}
extern "C" int mscl_adamw_step(const mscl_adamw_desc* d, void* stream) {
  if (!d || !d->tensors || !d->grads || !d->chunk_tensor || !d->m || !d->v || !d->words || !d->lr || d->n_chunks <= 0) return MSCL_E_ARG;
  if (!(d->beta1 >= 0 && d->beta1 < 1 && d->beta2 >= 0 && d->beta2 < 1)) return MSCL_E_ARG;
  if (!((float)d->eps >= FLT_MIN)) return MSCL_E_ARG;          // the reciprocal of a subnormal is infinite
  if (!(d->max_norm > 0 || d->max_norm <= 0)) return MSCL_E_ARG;          // NaN
  if (d->max_norm > 0 && (!d->partials || !d->grad_norm)) return MSCL_E_ARG;
  if (d->state_bits != 32 && d->state_bits != 8) return MSCL_E_SHAPE;
  if (d->state_bits == 8 && (!d->exponents || d->n_blocks <= 0)) return MSCL_E_ARG;
  if (d->shadow_type != MSCL_NONE && d->shadow_type != MSCL_BF16 && d->shadow_type != MSCL_F16) return MSCL_E_SHAPE;
  if (((uintptr_t)d->m | (uintptr_t)d->v) & 15) return MSCL_E_SHAPE;
  hipStream_t st = (hipStream_t)stream;
  switch (d->grad_type) {
    case MSCL_F32: return adamw_launch<MSCL_F32>(*d, st);
    case MSCL_BF16: return adamw_launch<MSCL_BF16>(*d, st);
    case MSCL_F16: return adamw_launch<MSCL_F16>(*d, st);
  }
  return MSCL_E_SHAPE;
}

// The values that 8-bit states stand for, as bf16 (exact: 4 significant bits, bf16 has 8).  A thread decodes 8 elements.  Bound by memory:
// 300 M elements, 1.8 GB, 345 us.  Non-temporal like the update (a step and its values at 32 / 300 M elements: 161 / 1169 us without, 154 / 1173 with).
__global__ __launch_bounds__(256) void adamw_values_kernel(const uint8_t* __restrict__ m, const uint8_t* __restrict__ v,
                                                           const uint8_t* __restrict__ ex, bf16_t* __restrict__ om, bf16_t* __restrict__ ov,
                                                           int64_t n_blocks) {
  for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < n_blocks * 32; q += (int64_t)gridDim.x * 256) {
    const uint2 a = ldnt((const uint2*)m + q), b = ldnt((const uint2*)v + q);
    const int Em = ex[q >> 5], Ev = ex[n_blocks + (q >> 5)];
    float fm[8], fv[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t ca = (i < 4 ? a.x : a.y) >> (8 * (i & 3)) & 255u, cb = (i < 4 ? b.x : b.y) >> (8 * (i & 3)) & 255u;
      fm[i] = Em == 255 ? __builtin_nanf("") : decode_m(ca, Em);
      fv[i] = Ev == 255 ? __builtin_nanf("") : decode_v(cb, Ev);
    }
    stnt((uint4*)om + q, pack8(fm));
    stnt((uint4*)ov + q, pack8(fv));
  }
}
extern "C" int mscl_adamw_values(const uint8_t* m, const uint8_t* v, const uint8_t* exponents, uint16_t* m_out, uint16_t* v_out,
                                 int64_t n_blocks, void* stream) {
  if (!m || !v || !exponents || !m_out || !v_out || n_blocks <= 0) return MSCL_E_ARG;
  if (((uintptr_t)m | (uintptr_t)v) & 7 || ((uintptr_t)m_out | (uintptr_t)v_out) & 15) return MSCL_E_SHAPE;
  int64_t blocks = cdiv64(n_blocks * 32, 256); if (blocks > 16384) blocks = 16384;
  hipLaunchKernelGGL(adamw_values_kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, m, v, exponents, m_out, v_out, n_blocks);
  MSCL_LAUNCH_CHECK();
  return 0;
}
