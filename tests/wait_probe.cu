// A wait that runs out, as a kernel's would (ring_ptx.cuh): on a barrier at which nobody arrives, for its second.  For test_gpu_status.py.
#include "../llama.cl_b200/csrc/ring_ptx.cuh"

namespace {

__global__ void wait_kernel(int* status, int code, int* failed) {
    __shared__ __align__(8) uint64_t bar;
    __shared__ int fail;
    fail = 0;
    q4fc::mbar_init(q4fc::smem_u32(&bar), 1);
    __syncthreads();
    q4fc::mbar_wait(q4fc::smem_u32(&bar), 0, &fail, status, code);
    *failed = fail;
}

}  // namespace

extern "C" int wait_probe(int* status, int code, int* failed, void* stream) {
    wait_kernel<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(status, code, failed);
    return (int)cudaGetLastError();
}
