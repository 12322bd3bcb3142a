// gpt2_w4_u4.hip — linear layers with 4-bit codes with zero points (gfx950).
#include "gpt2_w4_linear.h"

template void dfattn::w4::launch_linear_format<dfattn::w4::kU4>(const LinearArgs &, bool, uint32_t, float *, hipStream_t);
