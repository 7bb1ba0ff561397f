// The token objectives' kernels for float16 logits.
#include "token_objectives.inc"

template struct sttfe::Launch<sttfe::half_t>;
