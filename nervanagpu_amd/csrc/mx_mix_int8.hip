// the int8 half of mx_mix.hip, apart from it for the sake of parallel builds
#define NG_MX_MIX_FORMAT NG_MX_INT8
#include "mx_mix.hip"
