/* hip_stub.c with a device memory that copies read and write, and the kernel that takes a flag. stub_late is a report that arrives right
 * behind a copy from the device. */
#define hipModuleLaunchKernel plain_launch
#define hipMemcpy plain_memcpy
#define hipMemset plain_memset
#include "hip_stub.c"
#undef hipModuleLaunchKernel
#undef hipMemcpy
#undef hipMemset
#include <string.h>

unsigned stub_late;
void stub_report(unsigned why) { memcpy(dev, &why, sizeof why); }

int hipModuleLaunchKernel(void *f, unsigned gx, unsigned gy, unsigned gz, unsigned bx, unsigned by, unsigned bz, unsigned lds, void *st, void **args, void **extra) {
  if (!strcmp(f, "amdc_take_flag")) {
    unsigned *flag = *(unsigned **)args[0], *to = *(unsigned **)args[1];
    *to = *flag, *flag = 0;
  }
  return 0;
}
int hipMemcpy(void *to, const void *from, size_t n, int kind) {
  memcpy(to, from, n);
  if (stub_late) stub_report(stub_late), stub_late = 0;
  return 0;
}
int hipMemset(void *p, int v, size_t n) { return memset(p, v, n < sizeof dev ? n : sizeof dev), 0; }
