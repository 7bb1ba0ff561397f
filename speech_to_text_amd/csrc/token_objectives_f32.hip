// The token objectives' kernels for float32 logits.
#include "token_objectives.inc"

template struct sttfe::Launch<float>;
