// gpt2_w4_e2m1.hip — linear layers with e2m1 codes (gfx950).
#include "gpt2_w4_linear.h"

template void dfattn::w4::launch_linear_format<dfattn::w4::kE2M1>(const LinearArgs &, bool, uint32_t, float *, hipStream_t);
