/* The HIP runtime that does nothing (hip_stub.c), which keeps the delta rule's arguments of the last launch as well. */
#define hipModuleLaunchKernel hipModuleLaunchKernel_counted
#include "hip_stub.c"
#undef hipModuleLaunchKernel
#include <stdint.h>
#include "../../amd.c_amd/csrc/amdc_layout.h"

amdc_gdn_args stub_gdn;
int hipModuleLaunchKernel(void *f, unsigned gx, unsigned gy, unsigned gz, unsigned bx, unsigned by, unsigned bz, unsigned lds, void *s, void **args) {
  (void)gx, (void)gy, (void)gz, (void)bx, (void)by, (void)bz, (void)lds, (void)s;
  return stub_gdn = *(const amdc_gdn_args *)args[1], hipModuleLaunchKernel_counted(f);
}
size_t stub_gdn_at(int i) { return i == 0 ? stub_gdn.vs : i == 1 ? stub_gdn.ys : i == 2 ? stub_gdn.few : i == 3 ? stub_gdn.tabs : stub_gdn.packed; }
