// The attention over the 16-bit paged caches in f16 (kv16_attn.cuh).
#define KV16_TYPE __half
#include "kv16_launch.cuh"
