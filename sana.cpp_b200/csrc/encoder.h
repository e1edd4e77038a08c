// Launchers of the operators of the text encoder's blocks (include/sana_cuda.h states their
// definitions): residual RMSNorm, rotary positions with the append to a paged cache, and
// attention of a chunk of new tokens over that cache.
#pragma once

#include <cstddef>

#include "common.cuh"

namespace sana {

enum DType : int { kF32 = 0, kBf16 = 1, kE4M3 = 2 };

// What a kernel found in device data that the host could not check, recorded in the int beside
// the handle's error code (Engine::bad()): a word of its own, so that it does not end the
// bounded waits of other kernels.
enum BadInput : int {
    kBadPage = 1,      // a page number outside the pool, or a position behind the table
    kBadRows = 2,      // row_start outside [0, rows], or more new tokens than max_new
    kBadLength = 3,    // kv_len negative, above max_kv, or below the number of new tokens
};
const char* bad_input_message(int code);
__device__ __forceinline__ void record_bad(int* bad, int code) { atomicCAS(bad, 0, code); }

struct AddRmsNorm {
    const void* x;
    const void* residual;  // or null
    void* sum;             // or null
    const float* weight;   // or null
    void* out;
    float* scale;          // E4M3 outputs
    long long ldx, ldr, ldo, rows;
    int x_dtype, r_dtype, out_dtype, C, group;
    float offset, eps;
};
constexpr int kNormMaxChannels = 16384;
void add_rms_norm(const AddRmsNorm& p, int num_sms, cudaStream_t st);

// The batch of sana_paged_batch and the pool of sana_paged_cache, as the kernels take them.
struct PagedBatch {
    int S, rows, max_new, max_kv;
    const int* row_start;
    const int* kv_len;
    const int* table;
    long long table_stride;
    int table_width;
};
// Sequence s of a batch. `ok`: its lengths are in order and it has new tokens; otherwise nothing of it is computed or
// written. `report`: this thread records what is out of order.
struct Sequence {
    int row0, n_new, past;
    bool ok;
};
__device__ __forceinline__ Sequence batch_sequence(const PagedBatch& b, int s, bool report, int* bad) {
    Sequence q;
    q.row0 = b.row_start[s];
    const int end = b.row_start[s + 1], len = b.kv_len[s];
    // 64-bit differences: the inputs are unchecked
    const long long n = static_cast<long long>(end) - q.row0;
    const bool rows_ok = q.row0 >= 0 && n >= 0 && end <= b.rows && n <= b.max_new;
    const bool len_ok = len >= 0 && len <= b.max_kv && (n == 0 || len >= n);
    if (report && !(rows_ok && len_ok)) record_bad(bad, rows_ok ? kBadLength : kBadRows);
    q.ok = rows_ok && len_ok && n > 0;
    q.n_new = static_cast<int>(n);
    q.past = len - static_cast<int>(n);
    return q;
}
struct PagedCache {
    void* k;
    void* v;
    int dtype, pages, page_size, kv_heads, D;
    long long page_stride, token_stride, head_stride;
};

struct Rotary {
    const double* freq;
    int rotated;  // 0: nothing turns
    int interleaved;
    float magnitude;
};
struct RotaryRows {
    Rotary rot;
    int dtype, D, q_heads, kv_heads;
    long long rows, ldq, ldk, ldv;
    const void* q;
    void* q_out;
    const void* k;
    void* k_out;           // without append
    const void* v;         // with append
    const int* positions;  // without append
    PagedBatch batch;      // with append
    PagedCache cache;
    int* bad;
};
void rotary_rows(const RotaryRows& p, bool append, cudaStream_t st);

struct PageDivisor {  // division by the page size (or another number) as a product (pattn.cu)
    uint32_t magic;
    int shift;
};
struct PagedAttention {
    PagedBatch batch;
    PagedCache cache;
    const void* q;
    void* out;
    long long ldq, ldo;
    int q_heads, window, sinks;
    float scale, softcap;
    void* workspace;
    int* bad;
    int* err;  // the handle's error word (bounded waits)
    PageDivisor page_div;  // set by paged_attention
};
// Bytes of workspace of a call (0: none), and the call. The two take the same decisions from the
// same sizes.
size_t paged_attention_workspace(const PagedAttention& p, int num_sms);
void paged_attention(PagedAttention p, int num_sms, cudaStream_t st);

}  // namespace sana
