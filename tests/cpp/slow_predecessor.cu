// A kernel that lets the stream's next kernel start at once and then takes its time: what stands in front of a dependent
// launch when the work before it is long.  Waits for nothing but the clock, and has its steps counted too.
#include <cuda_runtime.h>

__global__ void slow_predecessor_kernel(unsigned long long ns) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  unsigned long long start, now;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(start));
  for (int i = 0; i < 10000000; ++i) {
    __nanosleep(1000);
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
    if (now - start >= ns) break;
  }
}

extern "C" int slow_predecessor(unsigned long long ns, cudaStream_t stream) {
  slow_predecessor_kernel<<<1, 1, 0, stream>>>(ns);
  return int(cudaGetLastError());
}
