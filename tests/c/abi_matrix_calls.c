/* The operators on a share's matrices from plain C11: workspaces and refusals,
 * host only. */
#include <stdio.h>

#include "suika_step.h"

int main(void) {
  static float data[128 * 128];
  const sr_ffn_shape s = {data, data, data, data, 4, 8, 16, 8, 8, 8, 16, SR_DT_F32, SR_ACT_GELU};
  uint64_t bytes = 0;
  int rc = sr_ffn_workspace(&s, 1, &bytes);
  printf("ffn %d %d\n", rc, bytes >= 4 * 16 * sizeof(float));
  sr_ffn_shape bad = s;
  bad.activation = 9;
  printf("activation %d\n", sr_ffn_workspace(&bad, 0, &bytes));
  const sr_ffn_grads grads = {data, NULL, NULL, NULL};
  rc = sr_ffn_grad_workspace(&s, data, 8, &grads, &bytes);
  printf("grad %d %d\n", rc, bytes > 0);
  const double coefficients[3] = {3.4445, -4.7750, 2.0315};
  sr_newton_schulz ns = {1, 0, coefficients, 1e-7, NULL, NULL};
  sr_matrix m = {data, 100, 120, 120, SR_DT_F32, -1};
  rc = sr_orthogonalize_workspace(&m, &m, 1, &ns, &bytes);
  printf("orthogonalize %d %d\n", rc, bytes > 0);
  m.split = 0;
  printf("split %d\n", sr_orthogonalize_workspace(&m, &m, 1, &ns, &bytes));
  ns.steps = 0;
  printf("steps %d\n", sr_orthogonalize_workspace(&m, &m, 0, &ns, &bytes));
  const sr_muon_options o = {1e-3, 0.1, 0.95, 1, 0, 0.0, NULL};
  ns.steps = 1;
  printf("muon %d %d\n", sr_muon(NULL, 0, &o, &ns, NULL, 0, NULL), sr_muon(NULL, 1, &o, &ns, NULL, 0, NULL));
  return 0;
}
