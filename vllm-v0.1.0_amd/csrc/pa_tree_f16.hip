// The kernels of pa_tree_kernel.h for one element type (a file of its own, so that the three compile in parallel).
#include "pa_tree_kernel.h"

int pa::tree_launch_f16(const TreeArgs& a, int head_size, unsigned grid, hipStream_t st) {
  return tree::tree_launch<tree::F16>(a, head_size, grid, st);
}
