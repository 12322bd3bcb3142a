// gpt2_w4_i4.hip — linear layers with int4 codes about 8 (gfx950).
#include "gpt2_w4_linear.h"

template void dfattn::w4::launch_linear_format<dfattn::w4::kI4>(const LinearArgs &, bool, uint32_t, float *, hipStream_t);
