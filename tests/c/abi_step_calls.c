/* The training-step operators' header from plain C11: workspaces and refusals,
 * host only. */
#include <stdio.h>

#include "suika_step.h"

int main(void) {
  float data[8] = {0};
  const sr_array arrays[2] = {{data, 8, SR_DT_F32, 0}, {data, 16, SR_DT_BF16, 0}};
  uint64_t bytes = 0;
  int rc = sr_square_sum_workspace(arrays, 2, &bytes);
  printf("sum %d %d\n", rc, bytes >= 16);
  const sr_array bad = {data, 8, SR_DT_I32, 0};
  printf("dtype %d\n", sr_square_sum_workspace(&bad, 1, &bytes));
  const int64_t tokens[3] = {0, 1, 2};
  const sr_embedding_shape e = {tokens, SR_DT_I64, SR_DT_F32, 3, 4, 5, 0, 1.0f, 0};
  bytes = 0;
  rc = sr_embedding_grad_workspace(&e, &bytes);
  printf("embedding %d %d\n", rc, bytes > 0);
  const sr_logprob_shape l = {data, tokens, SR_DT_I64, SR_DT_F32, 2, 4, 4, 4};
  printf("logprob %d\n", sr_logprob_workspace(&l, 4, &bytes));
  printf("top %d\n", sr_logprob_workspace(&l, 5, &bytes));
  const sr_adamw_options o = {1e-3, 0.9, 0.99, 1e-8, 0.1, 0, 1.0};
  rc = sr_adamw(NULL, 0, &o, NULL, NULL);
  printf("step %d %d\n", rc, sr_last_error()[0] != 0);
  return 0;
}
