// Drawing tokens from bf16 logits (a source of its own: they compile beside each other).
#include "sample.h"

template int ulm::smp::launch<ULM_BF16>(ulm::smp::Args, hipStream_t);
