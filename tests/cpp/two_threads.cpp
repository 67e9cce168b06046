// Two host threads that each repeat one rrr_attention_kv4 call on a context of their own, without
// an interpreter's lock between them. Returns the first status that is not RRR_OK.
#include <atomic>
#include <thread>

#include "../../include/rrr_cuda.h"

struct KV4Call {
  rrr_ctx* ctx;
  const rrr_kv4_cache* cache;
  int n_heads, type;
  const void* q;
  int64_t q_stride;
  const int32_t* kv_lens;
  void* out;
  int64_t out_stride;
  void* workspace;
  int64_t workspace_bytes;
  void* stream;
};

extern "C" int repeat_attention_kv4(decltype(&rrr_attention_kv4) attention, const KV4Call* calls, int times) {
  std::atomic<int> ready{0}, code{RRR_OK};
  auto repeat = [&](const KV4Call& c) {
    ++ready;
    while (ready.load() < 2) {
    }
    for (int i = 0; i < times && code.load() == RRR_OK; ++i) {
      const int rc = attention(c.ctx, c.cache, c.n_heads, c.type, c.q, c.q_stride, c.kv_lens, 0.f, c.out, c.out_stride,
                               c.workspace, c.workspace_bytes, c.stream);
      if (rc != RRR_OK) code = rc;
    }
  };
  std::thread other(repeat, std::cref(calls[1]));
  repeat(calls[0]);
  other.join();
  return code.load();
}
