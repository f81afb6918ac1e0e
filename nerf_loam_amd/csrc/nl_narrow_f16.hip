// nl_narrow_f16.hip -- the streaming product of nl_narrow.h for float16
#include "nl_narrow.h"

void nl_narrow_f16(const NlGemm& g, const NlDz& z, int act, bool b_slow, int dz, unsigned grid, hipStream_t st) { nl_narrow_launch<_Float16>(g, z, act, b_slow, dz, grid, st); }
