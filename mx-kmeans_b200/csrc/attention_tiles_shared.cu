// The attention kernels for many query rows, for calls whose sequences share prefixes.
#define MXK_ATTENTION_PARAMS SharedParams
#include "attention_tiles.cu"
