// The kernels that come after a scoring pass, on statistics and status words that the host has prepared: what they give
// when a device wait of the pass has expired.  (A wait that expires in earnest takes a GPU that has stopped answering.)
// Built by test_gpu_expired_wait.py against libmtp.so.
#include "lm_score.cu"

extern "C" int test_score_join(const int64_t *targets, float *part, float *hit, int *status, int ctas, int rows, int V,
                               int tiles_n, float *logprob, float *entropy, void *stream) {
  ScoreParams p{};
  p.targets = targets;
  p.part = part;
  p.hit = hit;
  p.status = status;
  p.M = rows;
  p.N = V;
  p.tiles_n = tiles_n;
  p.c2 = LOG2E;
  launch_pdl(lm_score_join_kernel<true>, dim3(ceil_div(rows, JOIN_ROWS)), dim3(32 * JOIN_WARPS), 0, (cudaStream_t)stream, p,
             ctas, 1.f, logprob, entropy);
  return check_launch("test_score_join");
}

// mtp_token_logprobs on fp32 logits [rows][V] that a product whose status word is `expired` has made.
extern "C" int test_rows_after_a_product(const float *logits, int64_t rows, int V, const int64_t *targets, float *logprob,
                                         float *entropy, int top_k, int64_t *top_ids, float *top_logprobs,
                                         const int *expired, void *stream) {
  return launch_token_logprobs(logits, MTP_F32, 1, rows, 0, V, V, targets, 1.f, logprob, entropy, nullptr, top_k, top_ids,
                               top_logprobs, expired, (cudaStream_t)stream);
}
