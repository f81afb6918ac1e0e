// nl_narrow_bf16.hip -- the streaming product of nl_narrow.h for bfloat16
#include "nl_narrow.h"

void nl_narrow_bf16(const NlGemm& g, const NlDz& z, int act, bool b_slow, int dz, unsigned grid, hipStream_t st) { nl_narrow_launch<__bf16>(g, z, act, b_slow, dz, grid, st); }
