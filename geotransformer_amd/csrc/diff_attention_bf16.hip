// diff_attention_bf16.hip -- the kernels of diff_attention.h for bf16 heads.
#include "diff_attention.h"

int geotr::dattn::launch_bf16(const Args& a, Which which, hipStream_t s) { return launch_type<__bf16>(a, which, s); }
