// The cross attention kernels of one element type.
#define ATTENTION_DEFINE_LAUNCHES
#include "attention.h"

ATTENTION_INSTANTIATE(bf16_t)
