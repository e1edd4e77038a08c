// Rotary positions, alone or with the append of a batch's keys and values to a paged cache.
//
// A turned pair is y_a = m (x_a cos t - x_b sin t), y_b = m (x_b cos t + x_a sin t) at the angle
// t = position * freq. Far positions would lose the angle in 32 bits (a position of 10^5 leaves
// 2^-7 radians of it), so the product is taken in 64 bits and reduced to a part of a turn there;
// the remaining |t| <= pi goes through sincospif. The angles of a row are the same for all its
// heads: the block computes them once into shared memory.
//
// One block per row. The kernel moves each q, k (and v) element once each way; what bounds it is
// HBM for many rows and launch plus latency for a decoding step. A row's lookups (sequence, length,
// page, frequencies) are four dependent loads: they are hidden by other rows, so blocks are small and
// hold few registers, 32 to an SM. 45000 rows of 16 + 4 heads of 128, bf16: 95 us, 5.9 TB/s (blocks
// of 128 threads 110, 32 of 64 without the bound on registers 119, elements fetched before the
// lookups, which takes registers, 132 to 154).
#include "encoder.h"

namespace sana {
namespace {

constexpr int kThreads = 64, kBlocksPerSm = 32;
constexpr int kMaxPairs = 256;  // head_dim <= 512

struct Args {
    RotaryRows p;
    int lo_units;  // units of the turned part per head (half layout: one unit is both sides)
    int units;     // all units of a head
};

// Sequence of a row: the number of sequences that end at or before it. All threads call it.
__device__ __forceinline__ int sequence_of(const int* row_start, int S, long long row) {
    int n = 0;
    for (int s0 = 0; s0 < S; s0 += kThreads) {
        const int s = s0 + static_cast<int>(threadIdx.x);
        n += __syncthreads_count(s < S && row_start[s + 1] <= row);
    }
    return n;
}

template <class T, int V>
struct alignas(sizeof(T) * V) Vec {
    T e[V];
};

// T element type; V elements per unit (16 bytes, or 1: pairs handled element by element at any
// alignment); IL interleaved pairs.
template <class T, int V, bool IL, bool APPEND>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) rotary_kernel(const __grid_constant__ Args a) {
    using U = Vec<T, V>;
    __shared__ float2 cs[kMaxPairs];
    const RotaryRows& p = a.p;
    const long long row = blockIdx.x;
    const int tid = threadIdx.x, D = p.D, pairs = p.rot.rotated / 2;
    int pos;
    long long place = -1;  // element offset of the token's place in the cache
    if constexpr (APPEND) {
        const int S = p.batch.S;
        // every sequence is checked by some block, its rows in the batch or not
        for (long long i = row + tid * p.rows; i < S; i += kThreads * p.rows) batch_sequence(p.batch, static_cast<int>(i), true, p.bad);
        const int s = sequence_of(p.batch.row_start, S, row);
        if (s >= S) return;  // behind the last sequence
        const Sequence sq = batch_sequence(p.batch, s, false, p.bad);
        // left out, in front of the first sequence, or of none that holds it (row_start not ascending)
        if (!sq.ok || row < sq.row0 || row - sq.row0 >= sq.n_new) return;
        pos = sq.past + static_cast<int>(row - sq.row0);
        const int slot = pos / p.cache.page_size;
        const int page = slot < p.batch.table_width ? p.batch.table[s * p.batch.table_stride + slot] : -1;
        if (page < 0 || page >= p.cache.pages) {
            if (tid == 0) record_bad(p.bad, kBadPage);
        } else {
            place = page * p.cache.page_stride + (pos - slot * p.cache.page_size) * p.cache.token_stride;
        }
    } else {
        pos = p.positions[row];
    }
    for (int i = tid; i < pairs; i += kThreads) {
        constexpr double kTurn = 0.15915494309189535;  // 1 / (2 pi)
        double t = static_cast<double>(pos) * p.rot.freq[i] * kTurn;
        t -= rint(t);
        float sn, cn;
        sincospif(2.0f * static_cast<float>(t), &sn, &cn);
        cs[i] = make_float2(cn * p.rot.magnitude, sn * p.rot.magnitude);
    }
    __syncthreads();

    const T* q = static_cast<const T*>(p.q) + row * p.ldq;
    T* q_out = static_cast<T*>(p.q_out) + row * p.ldq;
    const T* k = static_cast<const T*>(p.k) + row * p.ldk;
    const int turned_heads = p.q_heads + p.kv_heads, turned = turned_heads * a.units;
    const int copied = APPEND ? p.kv_heads * (D / V) : 0;
    for (int it = tid; it < turned + copied; it += kThreads) {
        if (it >= turned) {  // a vector of v
            const int c = it - turned, h = c / (D / V), d = (c - h * (D / V)) * V;
            if (place >= 0)
                *reinterpret_cast<U*>(static_cast<T*>(p.cache.v) + place + h * p.cache.head_stride + d) =
                    *reinterpret_cast<const U*>(static_cast<const T*>(p.v) + row * p.ldv + static_cast<long long>(h) * D + d);
            continue;
        }
        const int head = it / a.units, u = it - head * a.units;
        const bool is_q = head < p.q_heads;
        const int h = is_q ? head : head - p.q_heads;
        const T* src = (is_q ? q : k) + static_cast<long long>(h) * D;
        T* dst;
        if (is_q) {
            dst = q_out + static_cast<long long>(h) * D;
        } else if constexpr (APPEND) {
            if (place < 0) continue;
            dst = static_cast<T*>(p.cache.k) + place + h * p.cache.head_stride;
        } else {
            dst = static_cast<T*>(p.k_out) + row * p.ldk + static_cast<long long>(h) * D;
        }
        if (u >= a.lo_units) {  // behind the turned part
            const int d = p.rot.rotated + (u - a.lo_units) * V;
            *reinterpret_cast<U*>(dst + d) = *reinterpret_cast<const U*>(src + d);
        } else if constexpr (IL && V > 1) {
            const int d = u * V;
            U x = *reinterpret_cast<const U*>(src + d), y;
#pragma unroll
            for (int j = 0; j < V / 2; ++j) {
                const float2 c = cs[d / 2 + j];
                const float xa = to_f(x.e[2 * j]), xb = to_f(x.e[2 * j + 1]);
                y.e[2 * j] = from_f<T>(xa * c.x - xb * c.y);
                y.e[2 * j + 1] = from_f<T>(xb * c.x + xa * c.y);
            }
            *reinterpret_cast<U*>(dst + d) = y;
        } else {
            const int da = IL ? 2 * u : u * V, db = IL ? da + 1 : da + pairs;
            const U xa = *reinterpret_cast<const U*>(src + da), xb = *reinterpret_cast<const U*>(src + db);
            U ya, yb;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float2 c = cs[IL ? u : da + j];
                const float fa = to_f(xa.e[j]), fb = to_f(xb.e[j]);
                ya.e[j] = from_f<T>(fa * c.x - fb * c.y);
                yb.e[j] = from_f<T>(fb * c.x + fa * c.y);
            }
            *reinterpret_cast<U*>(dst + da) = ya;
            *reinterpret_cast<U*>(dst + db) = yb;
        }
    }
}

template <class T, int V, bool APPEND>
void launch(const RotaryRows& p, cudaStream_t st) {
    Args a;
    a.p = p;
    const int rest = (p.D - p.rot.rotated) / V;
    // half layout (and single elements): a unit is one vector on each side; interleaved vectors hold their own pairs
    a.lo_units = p.rot.interleaved && V > 1 ? p.rot.rotated / V : p.rot.rotated / 2 / V;
    a.units = a.lo_units + rest;
    const unsigned grid = static_cast<unsigned>(p.rows);
    if (p.rot.interleaved) rotary_kernel<T, V, true, APPEND><<<grid, kThreads, 0, st>>>(a);
    else rotary_kernel<T, V, false, APPEND><<<grid, kThreads, 0, st>>>(a);
    SANA_CUDA(cudaGetLastError());
}

template <class T, bool APPEND>
void by_alignment(const RotaryRows& p, cudaStream_t st) {
    constexpr int V = 16 / sizeof(T);
    bool vec = p.D % V == 0 && p.rot.rotated % (p.rot.interleaved ? V : 2 * V) == 0;
    auto ok = [&](const void* ptr, long long ld) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0 && ld % V == 0; };
    if (p.q_heads) vec = vec && ok(p.q, p.ldq) && ok(p.q_out, p.ldq);
    if (p.kv_heads) {
        vec = vec && ok(p.k, p.ldk);
        if (APPEND)
            vec = vec && ok(p.v, p.ldv) && ok(p.cache.k, p.cache.page_stride) && ok(p.cache.v, p.cache.token_stride) &&
                  p.cache.head_stride % V == 0;
        else
            vec = vec && ok(p.k_out, p.ldk);
    }
    if (vec) launch<T, V, APPEND>(p, st);
    else launch<T, 1, APPEND>(p, st);
}

}  // namespace

const char* bad_input_message(int code) {
    switch (code) {
        case kBadPage: return "a sequence's page number lies outside the pool, or a position behind its page table";
        case kBadRows: return "row_start is not ascending within the batch's rows, or a sequence has more than max_new new tokens";
        default: return "kv_len is negative, above max_kv, or below the sequence's new tokens";
    }
}

void rotary_rows(const RotaryRows& p, bool append, cudaStream_t st) {
    if (p.rows == 0) return;
    if (p.dtype == kF32) {
        if (append) by_alignment<float, true>(p, st);
        else by_alignment<float, false>(p, st);
    } else {
        if (append) by_alignment<bf16, true>(p, st);
        else by_alignment<bf16, false>(p, st);
    }
}

}  // namespace sana
