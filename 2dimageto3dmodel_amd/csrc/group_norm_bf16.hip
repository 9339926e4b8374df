// The group norm kernels of one element type (group_norm.h).
#include <type_traits>

#define M355_GN_T __bf16
#define M355_GN_RUN run_bf16
#include "group_norm_types.h"
