// Residual norm: argument checks, the plan of a launch, entry points.  The kernels are in res_norm.h; each pair of types is compiled in a
// translation unit of its own (res_norm_*.hip).
#include "res_norm.h"

#define TYPES(X, F) \
  extern template void res_norm_fwd_types<X, F>(const mscl_res_norm_desc&, hipStream_t); \
  extern template int res_norm_bwd_types<X, F>(const mscl_res_norm_desc&, const BwdPlan&, hipStream_t);
TYPES(MSCL_BF16, MSCL_BF16)
TYPES(MSCL_F16, MSCL_F16)
TYPES(MSCL_F32, MSCL_F32)
TYPES(MSCL_F32, MSCL_BF16)
TYPES(MSCL_F32, MSCL_F16)
#undef TYPES

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
// Lanes of a row: the fewest that hold it at 8 NV channels each -- a power of two up to 64, then whole waves.  (16 channels a lane in one wave
// for 513 .. 1024 channels: forward of 24 M elements bf16 / fp32 35.3 / 52.2 us at 1024, 33.9 / 49.6 us with two waves.)
void res_norm_team(int C, int* T, int* wave, int* nv) {
  *nv = 1;
  *wave = 1;
  for (int t = 1; t <= 64; t *= 2) if (C <= 8 * t) { *T = t; return; }
  *wave = 0;
  *nv = C > 8192 ? 2 : 1;
  const int need = (C + 8 * *nv - 1) / (8 * *nv);
  *T = (need + 63) / 64 * 64;
}
extern "C" int mscl_res_norm_fwd(const mscl_res_norm_desc* d, void* stream) {
  const int rc = res_norm_check(d);
  if (rc) return rc;
  if ((d->f && !d->y) || (d->pre && !d->h)) return MSCL_E_ARG;
  hipStream_t st = (hipStream_t)stream;
  if (d->x_type == MSCL_BF16) res_norm_fwd_types<MSCL_BF16, MSCL_BF16>(*d, st);
  else if (d->x_type == MSCL_F16) res_norm_fwd_types<MSCL_F16, MSCL_F16>(*d, st);
  else if (d->f_type == MSCL_F32) res_norm_fwd_types<MSCL_F32, MSCL_F32>(*d, st);
  else if (d->f_type == MSCL_BF16) res_norm_fwd_types<MSCL_F32, MSCL_BF16>(*d, st);
  else res_norm_fwd_types<MSCL_F32, MSCL_F16>(*d, st);
  MSCL_LAUNCH_CHECK();
  return 0;
}

static BwdPlan bwd_plan(const mscl_res_norm_desc* d) {
  BwdPlan p;
  res_norm_team(d->C, &p.T, &p.wave, &p.nv);
  const int per = p.wave ? 256 / p.T : 1;
  p.rows_per_gate = (int)(d->gate ? d->rows_per_gate : d->rows);
  p.gates = (int)(d->rows / p.rows_per_gate);
  // Many short runs: a team each.  (24 M elements, bf16, C = 64 / 512 / 2048, a training pass, WHOLE against SPLIT: runs of 8 rows 121 / 112 /
  // 114 against 725 / 208 / 150 us, 16 rows 113 / 110 / 113 against 398 / 151 / 129, 32 rows 131 / 119 / 118 against 233 / 123 / 117; 64 rows, C = 64 /
  // 192: 154 / 161 against 159 / 127.)  Few runs of any length leave most teams without one.
  // Past 8192 channels WHOLE has the most spills and is for very many gates alone (SPLIT's sums of each gate are 16 bytes a channel): 2000 x 12000
  // bf16, runs of 8 / 2 rows 467 / 578 us, SPLIT 294 / 399.
  const int teams = (p.wave ? 1024 : 4096 / (p.T / 64)) * per;
  const bool many = p.gates >= 4 * teams || (p.nv == 1 && p.rows_per_gate <= 32 && p.gates >= (teams / 2 < 1024 ? teams / 2 : 1024));
  p.mode = !d->gate ? SPLIT : p.rows_per_gate == 1 ? EACH1 : many ? WHOLE : SPLIT;
  // As many blocks as the 256 CUs hold at once (every block costs up to 4 C floats of column sums, and a second round of a few blocks as much
  // time as the first).
  const int waves = bwd_waves(p.wave ? 256 : p.T, d->x_type, d->f_type, p.mode, p.mode == WHOLE || d->b_post || d->b_pre || d->C < 8);
  const int target = 256 * (p.wave ? waves : waves * 4 / (p.T / 64));
  if (p.mode != SPLIT) {
    p.per_gate = 1;
    p.share = p.rows_per_gate;
    const int64_t need = cdiv64(p.gates, per);
    p.blocks = (int)(need < target ? need : target);
  } else {
    // blocks of a gate: the number with the fewest row times, rounds of the CUs times a team's rows and 3 for a block's column sums
    // (against the nearest number that fills them: 46800 x 512, 150 gates, bf16, a training pass 122 -> 108 us; 62300 x 64, 700 gates 44 -> 39)
    int64_t pg = 1, best = INT64_MAX;
    for (int rounds = 1; rounds <= 4; ++rounds) {
      const int64_t n = (int64_t)rounds * target / p.gates > 1 ? (int64_t)rounds * target / p.gates : 1;
      const int64_t cost = cdiv64(n * p.gates, target) * (cdiv64(cdiv64(p.rows_per_gate, n), per) + 3);
      if (cost < best) { best = cost; pg = n; }
    }
    p.share = (int)(cdiv64(cdiv64(p.rows_per_gate, pg), per) * per);             // whole rounds of the block's teams
    p.per_gate = (int)cdiv64(p.rows_per_gate, p.share);
    p.blocks = p.per_gate * p.gates;
  }
  return p;
}
extern "C" int64_t mscl_res_norm_ws(const mscl_res_norm_desc* d) {
  if (res_norm_check(d)) return 0;
  return (int64_t)bwd_plan(d).blocks * 4 * d->C;
}
extern "C" int mscl_res_norm_bwd(const mscl_res_norm_desc* d, void* stream) {
  const int rc = res_norm_check(d);
  if (rc) return rc;
  if (!d->dy && !d->dh) return MSCL_E_ARG;
  if ((d->db_post && !d->b_post) || (d->db_pre && !d->b_pre) || (d->dgate && !d->gate)) return MSCL_E_ARG;        // no sums are kept for these
  if ((d->dh && (!d->pre || !d->rstd_y || (d->pre == MSCL_NORM_LAYER && !d->mean_y)))) return MSCL_E_ARG;
  if (d->f && d->post && (!d->rstd_f || (d->post == MSCL_NORM_LAYER && !d->mean_f))) return MSCL_E_ARG;
  const BwdPlan p = bwd_plan(d);
  if (!d->ws || d->ws_floats < (int64_t)p.blocks * 4 * d->C) return MSCL_E_ARG;
  hipStream_t st = (hipStream_t)stream;
  if (d->x_type == MSCL_BF16) return res_norm_bwd_types<MSCL_BF16, MSCL_BF16>(*d, p, st);
  if (d->x_type == MSCL_F16) return res_norm_bwd_types<MSCL_F16, MSCL_F16>(*d, p, st);
  if (d->f_type == MSCL_F32) return res_norm_bwd_types<MSCL_F32, MSCL_F32>(*d, p, st);
  if (d->f_type == MSCL_BF16) return res_norm_bwd_types<MSCL_F32, MSCL_BF16>(*d, p, st);
  return res_norm_bwd_types<MSCL_F32, MSCL_F16>(*d, p, st);
}
