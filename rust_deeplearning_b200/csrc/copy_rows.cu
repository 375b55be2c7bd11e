// Rows of tensors copied within them: in tensors [sets][rows][...], row dst[i] of every set becomes row src[i] of that set, for several
// tensors and lists of rows in one launch (the pages and states of a cache, of all layer runs).
//
// Nothing but memory bounds it: 872 MB in keys and values of 26 layers copied in 257 us, 6.8 TB/s read and written (calls in a graph; a
// call among others 266); a page of 13 layers in 2.2 us, a launch and a trip to memory.  The description (where each tensor lies, which rows) travels in the kernel's parameters, so that
// nothing has to be copied to the device ahead of it and nothing in host memory has to outlive the call.
#include "api.h"
#include "common.cuh"
#include "launch.cuh"

static_assert(sizeof(CopyRowsTensor) == 48, "kernels/ops.py packs 48 bytes");

namespace {

constexpr int CR_THREADS = 256, CR_DEPTH = 8;                       // 16-byte vectors a thread has on their way
constexpr int CR_PIECE = CR_THREADS * CR_DEPTH * 16;                // bytes a block copies

struct CrTensor {
    char* base;
    long long set_stride, row_stride, row_bytes;    // bytes
    int pieces;                                     // of a row
    int first_pair, pairs;
    unsigned first_block;                           // blocks of the tensors before it
    int unit;                                       // what all of the above are multiples of: 16, 8, 4, 2 or 1
};

// CUDA passes up to 32,764 bytes; a short list costs the host less to pass
template <int PAIRS>
struct CrArgs {
    CrTensor tensor[RDL_COPY_ROWS_MAX_TENSORS];
    int n_tensors;
    int2 pair[PAIRS];                               // source row, destination row
};
constexpr int CR_FEW = 64, CR_MANY = 2048;
constexpr long long CR_MAX_BLOCKS = 0x7fffffff;     // of a launch
__host__ inline long long cr_pieces(const CopyRowsTensor& t) { return (t.row_bytes + CR_PIECE - 1) / CR_PIECE; }

template <typename U>
__device__ __forceinline__ void cr_copy(char* to, const char* from, int bytes) {
    const int n = bytes / (int)sizeof(U);
    for (int first = 0; first < n; first += CR_THREADS * CR_DEPTH) {
        U v[CR_DEPTH];
#pragma unroll
        for (int j = 0; j < CR_DEPTH; ++j) {
            const int i = first + j * CR_THREADS + (int)threadIdx.x;
            if (i < n) v[j] = __ldcs((const U*)from + i);
        }
#pragma unroll
        for (int j = 0; j < CR_DEPTH; ++j) {
            const int i = first + j * CR_THREADS + (int)threadIdx.x;
            if (i < n) __stcs((U*)to + i, v[j]);
        }
    }
}

template <int PAIRS>
__global__ void __launch_bounds__(CR_THREADS) copy_rows_kernel(const __grid_constant__ CrArgs<PAIRS> a) {
    int i = 0;
    while (i + 1 < a.n_tensors && blockIdx.x >= a.tensor[i + 1].first_block) ++i;
    const CrTensor& t = a.tensor[i];
    const unsigned block = blockIdx.x - t.first_block;
    const unsigned row = block / (unsigned)t.pieces, piece = block - row * (unsigned)t.pieces;
    const unsigned set = row / (unsigned)t.pairs;
    const int2 p = a.pair[t.first_pair + (int)(row - set * (unsigned)t.pairs)];
    char* at = t.base + set * t.set_stride + (long long)piece * CR_PIECE;
    const long long left = t.row_bytes - (long long)piece * CR_PIECE;
    const int bytes = (int)(left < CR_PIECE ? left : CR_PIECE);
    char* to = at + p.y * t.row_stride;
    const char* from = at + p.x * t.row_stride;
    rdl_grid_wait();
    rdl_grid_launch_dependents();
    switch (t.unit) {
        case 16: cr_copy<uint4>(to, from, bytes); break;
        case 8: cr_copy<uint2>(to, from, bytes); break;
        case 4: cr_copy<unsigned>(to, from, bytes); break;
        case 2: cr_copy<unsigned short>(to, from, bytes); break;
        default: cr_copy<unsigned char>(to, from, bytes); break;
    }
}

template <int PAIRS>
int cr_run(const CopyRowsTensor* tensors, int n_tensors, const int* pairs, cudaStream_t st) {
    // as many lists, or parts of lists, as fit the parameters go into one launch
    int i = 0, done = 0;                             // tensor, pairs of its list that have been launched
    while (i < n_tensors) {
        CrArgs<PAIRS> a;
        int used = 0;
        unsigned blocks = 0;
        a.n_tensors = 0;
        int last_whole = -1;
        for (; i < n_tensors; done == tensors[i].pairs ? (++i, done = 0) : 0) {
            const CopyRowsTensor& t = tensors[i];
            // a list that the tensor before brought whole is there already (keys and values move alike)
            const CrTensor* last = a.n_tensors ? &a.tensor[a.n_tensors - 1] : nullptr;
            const bool there = done == 0 && i > 0 && last && last_whole == i - 1 && tensors[i - 1].first_pair == t.first_pair && tensors[i - 1].pairs == t.pairs;
            const int room = PAIRS - used;
            if (!there && room == 0) break;
            const long long pieces = cr_pieces(t), of_row = pieces * t.sets;
            if (of_row == 0 || t.pairs == 0) { done = t.pairs; continue; }
            const long long fit = (CR_MAX_BLOCKS - blocks) / of_row;                 // rows that this launch has blocks for
            if (fit == 0) break;
            int take = there || t.pairs - done < room ? t.pairs - done : room;
            if (take > fit) take = (int)fit;
            const int fresh = there ? 0 : take, at = there ? last->first_pair : used;
            const uintptr_t all = (uintptr_t)t.base | (uintptr_t)t.set_stride | (uintptr_t)t.row_stride | (uintptr_t)t.row_bytes;
            CrTensor& c = a.tensor[a.n_tensors++];
            c = {(char*)t.base, t.set_stride, t.row_stride, t.row_bytes, (int)pieces, at, take, blocks, all & 15 ? (int)(all & (~all + 1)) : 16};
            const int *src = pairs + 2 * t.first_pair + done, *dst = src + t.pairs;
            for (int k = 0; k < fresh; ++k) a.pair[at + k] = make_int2(src[k], dst[k]);
            if (take == t.pairs) last_whole = i;
            used += fresh;
            blocks += (unsigned)(of_row * take);
            done += take;
        }
        if (blocks) RDL_CHECK_EX(rdl_launch(copy_rows_kernel<PAIRS>, dim3(blocks), dim3(CR_THREADS), 0, st, a), "copy_rows");
    }
    return 0;
}

}  // namespace

extern "C" int rdl_copy_rows(const CopyRowsTensor* tensors, int n_tensors, const int* pairs, void* stream) {
    RDL_REQUIRE(n_tensors >= 0 && n_tensors <= RDL_COPY_ROWS_MAX_TENSORS, "copy_rows: %d tensors, %d at most", n_tensors, RDL_COPY_ROWS_MAX_TENSORS);
    long long total = 0;
    for (int i = 0; i < n_tensors; ++i) {
        const CopyRowsTensor& t = tensors[i];
        RDL_REQUIRE(t.sets >= 0 && t.pairs >= 0 && t.row_bytes >= 0 && (t.base || !t.row_bytes || !t.pairs || !t.sets), "copy_rows: bad tensor %d", i);
        RDL_REQUIRE(cr_pieces(t) == 0 || t.sets <= CR_MAX_BLOCKS / cr_pieces(t), "copy_rows: tensor %d has rows that a launch has no blocks for", i);
        total += t.pairs;
    }
    RDL_REQUIRE(total == 0 || pairs, "copy_rows: missing list");
    return total <= CR_FEW ? cr_run<CR_FEW>(tensors, n_tensors, pairs, (cudaStream_t)stream)
                           : cr_run<CR_MANY>(tensors, n_tensors, pairs, (cudaStream_t)stream);
}
