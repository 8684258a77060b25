// The waits of the prompt kernels when one of them gives up, in the form of attn_stream_kernel: four consumer warps and one that
// requests.  Every wait is bounded; see test_gpu_wait_giveup.py.
#include "gdnr_tile.cuh"

using namespace gdnr;

namespace {

constexpr int WARPS = 4, WORDS = 4096, STAGES = 2;

struct Shared {
  alignas(128) uint32_t tile[STAGES][WORDS];
  uint64_t full[STAGES], never;
  int abort;
};

// report: what each consumer warp's own wait said, whether it left through the barrier, words that differ after the drain
__global__ void __launch_bounds__(WARPS * 32 + 32) giveup_kernel(const uint32_t* src, uint32_t* err, int* report) {
  extern __shared__ __align__(128) uint8_t raw[];
  Shared& sh = *reinterpret_cast<Shared*>(raw);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) mbar_init(&sh.full[i], 1);
    mbar_init(&sh.never, 1);
    sh.abort = 0;
    fence_mbar_init();
  }
  __syncthreads();
  if (warp == WARPS) {
    if (lane == 0)
      for (int i = 0; i < STAGES; ++i) {
        mbar_arrive_expect_tx(&sh.full[i], WORDS * 4);
        bulk_g2s(sh.tile[i], src + i * WORDS, WORDS * 4, &sh.full[i]);
      }
    __syncwarp();
    drain(sh.full, STAGES, STAGES);
    int differ = 0;
    for (int i = lane; i < STAGES * WORDS; i += 32) differ += (&sh.tile[0][0])[i] != src[i];
    differ = __reduce_add_sync(0xffffffffu, differ);
    if (lane == 0) report[2 * WARPS] = differ;
    return;
  }
  const WarpWait wait{err, &sh.abort};
  // the first warp's barrier is one that nothing arrives on; the others' tile lands
  const bool ok = wait(warp == 0 ? &sh.never : &sh.full[0], 0);
  if (lane == 0) report[warp] = ok;
  if (bar_or(1, WARPS * 32, !ok)) {
    if (lane == 0) report[WARPS + warp] = 1;
    return;
  }
  bar_sync(1, WARPS * 32);
}

}  // namespace

extern "C" int run(const uint32_t* src, uint32_t* err, int* report) {
  if (cudaFuncSetAttribute(giveup_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(sizeof(Shared))) != cudaSuccess) return 1;
  giveup_kernel<<<1, WARPS * 32 + 32, sizeof(Shared)>>>(src, err, report);
  return cudaGetLastError() != cudaSuccess;
}
