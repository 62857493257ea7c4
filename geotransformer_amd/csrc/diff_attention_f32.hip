// diff_attention_f32.hip -- the kernels of diff_attention.h for fp32 heads.
#include "diff_attention.h"

int geotr::dattn::launch_f32(const Args& a, Which which, hipStream_t s) { return launch_type<float>(a, which, s); }
