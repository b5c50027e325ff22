// The plans of block_norm and its gradients for every width: what a launch takes
// of shared memory is within what every launch asks for, at least two rows are
// on their way where rows are staged, and threads and groups cover the row.
#include <stdio.h>

#include "loom_b200_block_norm.cuh"

using namespace loomb;

static int bad(int line, int width, const RowPlan& s) {
  fprintf(stderr, "line %d: width %d, stages %d, threads %u, per %d, shared %zu\n", line, width,
          s.stages, s.threads, s.per, s.shared);
  return 1;
}

template <class Tx, class Tb>
static int check(int width, bool phased) {
  const RowPlan plans[] = {
      row_plan(width, phased, true, ForwardStage<Tx, Tb>::words, 0, 512, 2, false),
      row_plan(width, phased, false, 0, 0, 1024, 1, false),
      row_plan(width, phased, true, GradStage<Tx, Tb>::words, 2 * GroupWords<Tb>::value, 512, 1,
               true),
      row_plan(width, phased, true, GradStage<Tx, Tb>::words, 2 * GroupWords<Tb>::value, 512, 2,
               true)};
  for (const RowPlan& s : plans) {
    const int phase = s.phased && width % 8 != 0 ? 7 : 0;
    if (s.shared > kStageBytes) return bad(__LINE__, width, s);
    if (s.stages != 0 && (s.stages < 2 || s.stages > 4)) return bad(__LINE__, width, s);
    if (s.stages == 0 && s.shared != 0) return bad(__LINE__, width, s);
    if ((int)s.threads * (s.warp ? kRowWarps : 1) > s.most) return bad(__LINE__, width, s);
    if ((int)s.threads * s.per * 8 < width + phase) return bad(__LINE__, width, s);
    if (!s.edge && ((int)s.threads * s.per * 8 != width) && s.stages != 0)
      return bad(__LINE__, width, s);
  }
  return 0;
}

int main() {
  for (int width = 1; width <= kRowMaxWidth; ++width)
    for (int phased = 0; phased < 2; ++phased)
      if (check<float, float>(width, phased) || check<float, __nv_bfloat16>(width, phased) ||
          check<__half, __half>(width, phased))
        return 1;
  printf("row plans ok\n");
  return 0;
}
