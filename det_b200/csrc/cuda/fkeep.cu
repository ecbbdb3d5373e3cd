// The accepted nodes of every tree become cached rows (include/det_b200.h, det_fkeep_op): rows move towards the front of the same
// cache.  A thread owns one 16-byte column of a cache and moves its pieces in order of the destination, eight at a time: the list
// ascends strictly, so source i is never before destination i, and a later source never lies among the destinations already
// written; no thread touches another's column, so nothing has to be waited for.  Bound by latency (list, then rows, then stores): 2.8 us for
// one path of 5 rows of 4 KB, 3.8 us for 32 sequences' in 8 layers.
#include "ftree.cuh"
#include <algorithm>

namespace detb {

struct KeepArgs {
    int layers, seqs, cap, pieces;      // 16-byte pieces of a row
    const det_seq_slot* table;
    const int* len;
    const int* keep;
    int keep_ld;
    const int* count;
    int max_count;
    int* len_out;
    int* error_flag;
};
constexpr int KEEP_THREADS = 128, KEEP_RUN = 8;

// grid (caches, pieces of a row)
__global__ void __launch_bounds__(KEEP_THREADS) k_fkeep(const KeepArgs a) {
    __shared__ int list[DET_MAX_TREE];
    pdl_trigger();
    pdl_wait();
    const int e = blockIdx.x, b = e % a.seqs, len = a.len[b];
    int n = a.count[b];
    bool fits = len >= 0 && n >= 0 && n <= a.max_count && len <= a.cap;
    // the caches of all layers of the sequence (a thread's first one is asked for ahead of the list): its blocks agree, and none moves rows when
    // one of them cannot
    bool usable = (int)threadIdx.x >= a.layers || usable_cache(a.table[b + (int)threadIdx.x * a.seqs].cache);
    if (fits)
        for (int i = threadIdx.x; i < n; i += KEEP_THREADS) {
            const int k = a.keep[(size_t)b * a.keep_ld + i];
            list[i] = k;
            if (k < i || k >= a.cap - len || (i > 0 && a.keep[(size_t)b * a.keep_ld + i - 1] >= k)) fits = false;
        }
    for (int i = threadIdx.x + KEEP_THREADS; i < a.layers; i += KEEP_THREADS) usable = usable && usable_cache(a.table[b + i * a.seqs].cache);
    fits = __syncthreads_and(fits && (usable || n == 0));      // with nothing to move the caches need not be there (a place not in use)
    if (!fits) {
        if (threadIdx.x == 0) report_size(a.error_flag);
        n = 0;
    }
    if (fits && a.len_out && e < a.seqs && blockIdx.y == 0 && threadIdx.x == 0) a.len_out[b] = len + n;
    const int c = blockIdx.y * KEEP_THREADS + threadIdx.x;
    if (c >= a.pieces) return;
    uint4* rows = static_cast<uint4*>(a.table[e].cache) + (size_t)len * a.pieces + c;
    for (int i0 = 0; i0 < n; i0 += KEEP_RUN) {
        uint4 v[KEEP_RUN];
#pragma unroll
        for (int j = 0; j < KEEP_RUN; j++)
            if (i0 + j < n) v[j] = rows[(size_t)list[i0 + j] * a.pieces];
#pragma unroll
        for (int j = 0; j < KEEP_RUN; j++)
            if (i0 + j < n && list[i0 + j] != i0 + j) rows[(size_t)(i0 + j) * a.pieces] = v[j];
    }
}

}  // namespace detb

using namespace detb;

extern "C" int det_f_tree_keep(const det_fkeep_op* op, cudaStream_t st) {
    const char* name = "det_f_tree_keep";
    DETB_TAKE(op != nullptr, "no descriptor");
    DETB_TAKE(op->caches >= 0 && op->seqs >= 0 && op->cap > 0 && op->max_count >= 0 && op->keep_ld >= op->max_count, "bad sizes");
    DETB_TAKE(op->max_count <= DET_MAX_TREE, "the tree is too large");
    DETB_TAKE(op->row_bytes > 0 && op->row_bytes % 16 == 0 && op->row_bytes <= 64 << 20, "rows must be whole 16-byte pieces");
    if (op->caches == 0 || op->seqs == 0) return 0;
    DETB_TAKE(op->caches % op->seqs == 0, "caches must be whole layers");
    DETB_TAKE(op->table && op->len && op->count && (op->keep || op->max_count == 0), "table, len, keep or count is NULL");
    DETB_TAKE(op->len_out != op->len, "len_out must not be len");
    DETB_TAKE(runtime_ready(), "no usable device");
    KeepArgs a{op->caches / op->seqs, op->seqs, op->cap, op->row_bytes / 16, op->table, op->len, op->keep, op->keep_ld, op->count, op->max_count, op->len_out, error_word()};
    const int pieces = (a.pieces + KEEP_THREADS - 1) / KEEP_THREADS;
    DETB_TAKE(pieces <= 65535, "the row is too long");
    return launched(name, launch_pdl_try(k_fkeep, dim3(op->caches, pieces), dim3(KEEP_THREADS), 0, queue_of(st), 1, a));
}
