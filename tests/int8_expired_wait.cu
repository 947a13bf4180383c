// The tensor-core forms of the int8 product with a short limit and copies that bring fewer bytes than the kernel waits for (boxes
// of half as many rows of a), so that its waits expire while nothing else is wrong: what it gives then, and that it returns.
// Built by test_gpu_int8_expired_wait.py against libmtp.so.
#include "int8_tc.cu"

using namespace mtp::i8;

// form 0: K over a cluster of `split` CTAs; 1 and 2: tiles of one CTA or of a pair, bn columns wide.  out is bf16.
extern "C" int test_int8_linear(int form, int split, int bn, int lose, unsigned long long timeout_ns, const int8_t *a, int64_t ld_a,
                                const float *a_scale, int M, int K, const int8_t *w, int64_t ld_w, const float *w_scale, int N,
                                void *out, int64_t ld_out, void *stream) {
  const Out o{out, ld_out, MTP_BF16, a_scale, w_scale, nullptr, 0};
  cudaStream_t s = (cudaStream_t)stream;
  CUtensorMap ta, tb, tc;
  memset(&tc, 0, sizeof(tc));
  const int cg = form == 2 ? 2 : 1;
  if (form == 0) {
    SplitParams p = split_params(M, K, N, o, split, bn);
    p.timeout_ns = timeout_ns;
    int rc = map_codes(&ta, a, M, K, ld_a, lose ? p.a_rows / 2 : p.a_rows);
    if (!rc) rc = map_codes(&tb, w, N, K, ld_w, p.bn);
    return rc ? rc : launch_split(ta, tb, p, s);
  }
  Params p = form == 1 ? tile_params<1>(M, K, N, o, bn) : tile_params<2>(M, K, N, o, bn);
  p.timeout_ns = timeout_ns;
  int rc = map_codes(&ta, a, M, K, ld_a, lose ? BM / 2 : BM);
  if (!rc) rc = map_codes(&tb, w, N, K, ld_w, bn / cg);
  if (!rc && p.tma_cols) rc = map_out(&tc, o, M, N);
  if (rc) return rc;
  return form == 1 ? launch<1, __nv_bfloat16>(ta, tb, tc, p, s) : launch<2, __nv_bfloat16>(ta, tb, tc, p, s);
}
