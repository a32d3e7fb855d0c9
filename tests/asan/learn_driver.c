/* Host code of the policy operators' C entries (argument checks, launch plans, the overlap test)
 * under AddressSanitizer + UBSan, with exactly sized host arrays; every call is refused or has
 * no work, so nothing needs a GPU. */
#include <math.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include "mev.h"

#define CHECK(x)                                                 \
  do {                                                           \
    if (!(x)) {                                                  \
      printf("FAILED line %d: %s\n", __LINE__, #x);              \
      return 1;                                                  \
    }                                                            \
  } while (0)

int main(void) {
  /* workspaces of many shapes: sizes, dtypes, few and many rows */
  const int32_t sizes[] = {1, 2, 7, 8, 13, 17, 24, 25, 33, 64, 65, 300, 1000, 2048, 5000, 20000,
                           40000, 98304, 98400, 131072, 1 << 20, 0x7fffffff};
  const int64_t rows[] = {0, 1, 2, 31, 256, 10240, 1 << 20, (int64_t)1 << 33};
  for (size_t i = 0; i < sizeof(sizes) / sizeof(sizes[0]); ++i)
    for (size_t j = 0; j < sizeof(rows) / sizeof(rows[0]); ++j)
      for (int d = MEV_F32; d <= MEV_F16; ++d) {
        mev_policy a;
        memset(&a, 0, sizeof(a));
        float loss;
        a.rows = rows[j];
        a.actions = sizes[i];
        a.dtype = d;
        CHECK(mev_policy_workspace(&a) >= 0);
        a.loss = &loss;
        CHECK(mev_policy_workspace(&a) >= 0);
      }
  mev_policy a;
  memset(&a, 0, sizeof(a));
  CHECK(mev_policy_workspace(&a) == MEV_EINVAL); /* no actions */
  a.actions = 4;
  a.action_bytes = 8;
  a.dtype = 3;
  CHECK(mev_policy_rows(&a, NULL) == MEV_EINVAL);
  a.dtype = MEV_BF16;
  CHECK(mev_policy_rows(&a, NULL) == MEV_OK); /* no rows, nothing asked */
  a.rows = 3;
  CHECK(mev_policy_rows(&a, NULL) == MEV_EINVAL); /* no logits */
  CHECK(mev_policy_rows(NULL, NULL) == MEV_EINVAL);

  mev_advantages v;
  memset(&v, 0, sizeof(v));
  CHECK(mev_advantages_run(&v, NULL) == MEV_OK);
  const int64_t ts[] = {1, 20, 33, 5000, 1 << 20}, cs[] = {1, 3, 70, 4096, 1 << 20};
  for (size_t i = 0; i < 5; ++i)
    for (size_t j = 0; j < 5; ++j) {
      v.T = ts[i];
      v.E = cs[j];
      v.U = 1 + (int64_t)(j % 2) * 29;
      CHECK(mev_advantages_workspace(&v) >= 0);
      CHECK(mev_advantages_run(&v, NULL) == MEV_EINVAL); /* no buffers */
    }
  v.E = (int64_t)1 << 41;
  CHECK(mev_advantages_workspace(&v) == MEV_EINVAL);
  CHECK(mev_advantages_workspace(NULL) == MEV_EINVAL);

  /* clipping: overlapping and bad buffers (the pointers are never read) */
  for (int32_t n = 1; n < 300; n += 37) {
    const void** src = malloc(n * sizeof(*src));
    void** dst = malloc(n * sizeof(*dst));
    int64_t* num = malloc(n * sizeof(*num));
    int32_t* dt = malloc(n * sizeof(*dt));
    float norm;
    for (int32_t i = 0; i < n; ++i) {
      src[i] = dst[i] = (char*)0x100000 + 1024 * i;
      num[i] = 257; /* 1,028 bytes: into its neighbour */
      dt[i] = MEV_F32;
    }
    const int64_t need = mev_clip_norm_workspace(num, n);
    CHECK(need > 0);
    if (n > 1) CHECK(mev_clip_norm(src, dst, num, dt, n, 1.0f, &norm, &norm, need, NULL) == MEV_EINVAL);
    CHECK(mev_clip_norm(src, dst, num, dt, n, NAN, &norm, &norm, need, NULL) == MEV_EINVAL);
    CHECK(mev_clip_norm(src, dst, num, dt, n, 1.0f, &norm, &norm, need - 1, NULL) == MEV_EINVAL);
    num[n - 1] = -1;
    CHECK(mev_clip_norm_workspace(num, n) == MEV_EINVAL);
    num[n - 1] = INT64_MAX;
    CHECK(mev_clip_norm_workspace(num, n) == MEV_EINVAL);
    free(src);
    free(dst);
    free(num);
    free(dt);
  }
  CHECK(mev_clip_norm_workspace(NULL, 3) == MEV_EINVAL);
  CHECK(mev_clip_norm_workspace(NULL, -1) == MEV_EINVAL);
  printf("ok\n");
  return 0;
}
