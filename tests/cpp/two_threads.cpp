// Two host threads that each repeat one call of an entry point on a context of their own, without
// an interpreter's lock between them. Returns the first status that is not RRR_OK.
#include <atomic>
#include <functional>
#include <thread>

#include "../../include/rrr_cuda.h"

template <typename Call, typename Make>
static int repeat(const Call* calls, int times, Make make) {
  std::atomic<int> ready{0}, code{RRR_OK};
  auto run = [&](const Call& c) {
    ++ready;
    while (ready.load() < 2) {
    }
    for (int i = 0; i < times && code.load() == RRR_OK; ++i) {
      const int rc = make(c);
      if (rc != RRR_OK) code = rc;
    }
  };
  std::thread other(run, std::cref(calls[1]));
  run(calls[0]);
  other.join();
  return code.load();
}

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
  return repeat(calls, times, [&](const KV4Call& c) {
    return attention(c.ctx, c.cache, c.n_heads, c.type, c.q, c.q_stride, c.kv_lens, 0.f, c.out, c.out_stride,
                     c.workspace, c.workspace_bytes, c.stream);
  });
}

struct GemmCall {  // W [n, k] times the m rows of x
  rrr_ctx* ctx;
  const void* w;
  const void* x;
  float* y;
  int m, k, n, qtype;
  void* stream;
};
extern "C" int repeat_gemm_kq_tc(decltype(&rrr_gemm_kq_batched_path) gemm, const GemmCall* calls, int times) {
  return repeat(calls, times, [&](const GemmCall& c) {
    return gemm(c.ctx, c.qtype, c.w, static_cast<const uint16_t*>(c.x), c.y, c.m, c.k, c.n, nullptr, RRR_GEMM_TCGEN05,
                c.stream);
  });
}
extern "C" int repeat_logits(decltype(&rrr_logits_f32_batched) logits, const GemmCall* calls, int times) {
  return repeat(calls, times, [&](const GemmCall& c) {
    return logits(c.ctx, static_cast<const float*>(c.w), static_cast<const float*>(c.x), c.y, c.y, c.m, c.n, c.k,
                  nullptr, 0.f, c.stream);
  });
}
