// Launches of the few-query items (few_item.h) from a step's work list: rows of drafted tokens, and decode rows whose GQA
// group is not 1, 2 or 4 query heads.
#include "few_item.h"

namespace lv {

template <typename T, int D, int NB, FewSets SETS>
__global__ __launch_bounds__(64 * kWaves, 2) void few_list_kernel(AttnParams p) {
  __shared__ __attribute__((aligned(16))) char smem[kWaves * kFewStages * kFewStage];
  constexpr int HP = SETS == kTwoHeads ? 2 : 1;
  const int ny = p.hkv / HP, bx = blockIdx.x / ny, kh = blockIdx.x - bx * ny;
  const DecodeWork w = decode_work(p, bx);
  if (bx >= w.count) return;
  few_item<T, D, NB, SETS>(p, w.row, w.split, w.per, kh * HP, smem);
}

template <typename T, int D>
static void launch_rows(const AttnParams& p, int query_rows, int hp, int items, hipStream_t stream) {
  const dim3 grid(items * (p.hkv / hp)), block(64 * kWaves);
  if (query_rows > 32)
    hipLaunchKernelGGL((few_list_kernel<T, D, (D == 64 ? 4 : 2), (D == 64 ? kOneSet : kTwoBlocks)>), grid, block, 0,
                       stream, p);
  else if (query_rows > 16 && hp == 2)
    hipLaunchKernelGGL((few_list_kernel<T, D, 2, kTwoHeads>), grid, block, 0, stream, p);
  else if (query_rows > 16)
    hipLaunchKernelGGL((few_list_kernel<T, D, 2, kOneSet>), grid, block, 0, stream, p);
  else if (hp == 2)
    hipLaunchKernelGGL((few_list_kernel<T, D, 1, kTwoHeads>), grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL((few_list_kernel<T, D, 1, kOneSet>), grid, block, 0, stream, p);
}

void launch_few_query(const AttnParams& p, int d, int query_rows, int hp, int dtype, int items, hipStream_t stream) {
  if (dtype == LV_DTYPE_BF16) {
    if (d == 64) launch_rows<BF16, 64>(p, query_rows, hp, items, stream);
    else launch_rows<BF16, 128>(p, query_rows, hp, items, stream);
  } else {
    if (d == 64) launch_rows<F16, 64>(p, query_rows, hp, items, stream);
    else launch_rows<F16, 128>(p, query_rows, hp, items, stream);
  }
}

}  // namespace lv
