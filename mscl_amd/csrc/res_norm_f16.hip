#include "res_norm.h"
template void res_norm_fwd_types<MSCL_F16, MSCL_F16>(const mscl_res_norm_desc&, hipStream_t);
template int res_norm_bwd_types<MSCL_F16, MSCL_F16>(const mscl_res_norm_desc&, const BwdPlan&, hipStream_t);
