// The token objectives' kernels for bfloat16 logits.
#include "token_objectives.inc"

template struct sttfe::Launch<sttfe::bf16_t>;
