// diff_attention_f16.hip -- the kernels of diff_attention.h for fp16 heads.
#include "diff_attention.h"

int geotr::dattn::launch_f16(const Args& a, Which which, hipStream_t s) { return launch_type<_Float16>(a, which, s); }
