// The host side of the entry points that serve several sequences (zh_serving.cpp) without a device, beside that of the
// long-context ones, whose stand-ins it shares.
#include "longctx_host.cpp"

#include "../../ziggy-llm_amd/csrc/zh_serving.cpp"

namespace zh {
hipError_t launch_head_rows(const HeadRows &, int, hipStream_t) { return launches++, hipSuccess; }
hipError_t launch_kv4_load(const Kv4Layer &, const Batch &, float *, float *, hipStream_t) { return launches++, hipSuccess; }
hipError_t launch_kv4_attention(const Kv4Attn &, int, hipStream_t) { return launches++, hipSuccess; }
hipError_t launch_token_logprobs(const TokenLogprobs &, int, hipStream_t) { return launches++, hipSuccess; }
}  // namespace zh
