// Drawing tokens from fp32 logits (a source of its own: they compile beside each other).
#include "sample.h"

template int ulm::smp::launch<ULM_F32>(ulm::smp::Args, hipStream_t);
