// How the work of a product with a 4-bit weight is divided.
#include <atomic>

#include "launch.cuh"
#include "mx_tensor.cuh"

namespace { __global__ void __launch_bounds__(576, 1) cluster_probe_kernel() {} }      // stands for a block of the products; never launched

// Clusters of `size` blocks, each block with a multiprocessor to itself, that run at the same time on the current device.  Fewer than
// multiprocessors / size: a cluster lies within one group of them, and what is left of a group stays empty (18 clusters of 8 on 148
// multiprocessors took two turns, 14 us where one took 6).
static int clusters_at_once(int size) {
    static std::atomic<int> known[64][9];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    if (const int k = known[dev][size].load(std::memory_order_relaxed)) return k - 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(size * 32);
    cfg.blockDim = dim3(576);
    cfg.dynamicSmemBytes = 200 * 1024;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (rdl_allow_shared<cluster_probe_kernel>(200 * 1024) != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, cluster_probe_kernel, &cfg) != cudaSuccess) {
        cudaGetLastError();                                  // an answer of none is safe: the tile is not shared
        n = 0;
    }
    known[dev][size].store(n + 1, std::memory_order_relaxed);
    return n;
}


int mx_split(int tiles, int blocks, int sms) {
    if (tiles * 2 > sms) return 1;
    for (int split = 8; split > 1; --split)
        if (blocks >= 2 * split && tiles <= clusters_at_once(split)) return split;
    return 1;
}

// Up to 128 rows: whether the kernel with the weight tile on the M side of its products is the faster one.  Both estimates are a block
// of columns' time in a row times how many follow one another; the first adds what a row's sums cost on their way out of a
// tile.  Measured, first against second (rows, columns, outputs): 17 x 2,304 x 4,096 6.3 against 9.8 us; 128 x 2,304 x 4,096 10.4, 10.8;
// 128 x 1,024 x 8,192 10.9, 7.8; 64 x 14,336 x 3,584 12.9, 38.3; 128 x 14,336 x 3,584 15.8, 39.0.
bool mx_some_rows_pay(const Mx4Matrix& w, int m) {
    const int sms = rdl_sm_count(), split = mx_split(w.tiles, w.blocks, sms), turns = split > 1 ? 1 : (w.tiles + sms - 1) / sms;
    const float some = 0.25f * (float)((w.blocks + split - 1) / split * turns) + 0.045f * (float)(m * turns);
    const float many = 0.33f * (float)(w.blocks * (((w.tiles + 1) / 2 + sms - 1) / sms));
    return some < many;
}
