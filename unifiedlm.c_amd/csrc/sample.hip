// Drawing tokens: the entry (the kernels: sample.h).
#include "sample.h"

using namespace ulm;

extern "C" int ulm_sample_tokens(const void *logits, int dtype, long long rows, long long inner, long long outer_stride,
                                 long long row_stride, int V, const void *u, int u_double, const ulm_sampling *how,
                                 long long *token, float *logprob, long long *kept, void *stream) {
    ULM_REQUIRE(rows >= 1 && rows <= (1LL << 34) && inner >= 1 && V >= 1 && V <= smp::kMaxV,
                "ulm_sample_tokens: bad sizes rows=%lld inner=%lld V=%d", rows, inner, V);
    ULM_REQUIRE(valid_dtype(dtype), "ulm_sample_tokens: bad dtype %d", dtype);
    ULM_REQUIRE(logits && u && how && token && logprob && kept, "ulm_sample_tokens: null pointer");
    int log_v = 0;
    while ((1 << log_v) < V) ++log_v;
    const smp::Args a{{static_cast<const char *>(logits), inner, outer_stride, row_stride, rows, V},
                      u,
                      {how->temperature, how->temperatures},
                      {how->top_p, how->top_ps},
                      {how->min_p, how->min_ps},
                      how->top_k,
                      how->top_ks,
                      token,
                      kept,
                      logprob,
                      u_double,
                      log_v <= 15 ? 47 : 62 - log_v,
                      0};
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (dtype == ULM_F32) return smp::launch<ULM_F32>(a, s);
    if (dtype == ULM_BF16) return smp::launch<ULM_BF16>(a, s);
    return smp::launch<ULM_F16>(a, s);
}
