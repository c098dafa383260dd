// The attention over the 16-bit paged caches in bf16 (kv16_attn.cuh).
#define KV16_TYPE __nv_bfloat16
#include "kv16_launch.cuh"
