// Attention of a chunk of new tokens over a paged cache:
//   out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),  s_j = scale q.k_j or cap tanh(scale q.k_j / cap),
// in one pass over the keys with the running maximum m and sum; scores, statistics and sums fp32.
// Two kernels here: a tensor-core one for bf16 (mma.sync; single tokens and short chunks, which
// read much and compute little) and a CUDA-core one for fp32 and for what the first does not take;
// pattn_tc.cu has the one for chunks that fill 128-row tiles.
// pattn.cuh has the packing of rows, the key ranges and the splits.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "pattn.cuh"
#include "tma.h"

namespace sana {
namespace pattn {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -INFINITY;

// --- CUDA cores -------------------------------------------------------------------------------
// 32 packed rows x 32 keys per step, four threads per row: thread c of a row takes keys c + 4 i of
// the scores and channels 4 c + 16 i of the output; for the copies, thread c of key tid / 4 takes the
// same channels of that key. q, k and v sit in shared memory as fp32 rows padded by four words, so
// that the eight rows (or four keys) a warp reads at once lie in different banks. fp32 keys and
// values come by cp.async a tile ahead (16 bytes each where rows are aligned, else 4); bf16 ones, of
// odd sizes or alignment only, are converted on the way. DM: channels that registers hold. 4 prompts
// of 8 to 120 tokens, 6 heads of 72 over 2, fp32: 35 us, bound by the latency of the shared-memory reads.
constexpr int kSRows = 32, kSKeys = 32, kSThreads = 128;

__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <class T, int DM>
__global__ void __launch_bounds__(kSThreads) paged_simt_kernel(const __grid_constant__ Args a, const int vec) {
    extern __shared__ float sm[];
    __shared__ int there[2][kSKeys];
    const PagedAttention& p = a.p;
    const int tid = threadIdx.x, D = p.cache.D, D4 = (D + 3) & ~3, ld = D4 + 4;
    float* Qs = sm;
    float* kv = Qs + kSRows * ld;  // [2][k, v][kSKeys][ld]
    const int tile = a.row_tiles - 1 - static_cast<int>(blockIdx.x % a.row_tiles);
    const int rest = blockIdx.x / a.row_tiles, split = rest % a.splits, s = rest / a.splits, kvh = blockIdx.y;
    cudaTriggerProgrammaticLaunchCompletion();  // the join's blocks may take their places
    const Sequence sq = sequence(p, s, blockIdx.x % (a.row_tiles * a.splits) == 0 && kvh == 0 && tid == 0);
    const int rr0 = tile * kSRows, n_rows = sq.n_new * a.G;
    if (!sq.ok || rr0 >= n_rows) return;
    const KeyTiles kt = key_tiles(sq.past, sq.n_new, a.G, rr0, rr0 + kSRows, p.window, p.sinks, kSKeys, a.align);
    const int t0 = split * a.split_tiles, t1 = min(kt.n, t0 + a.split_tiles);
    if (t0 >= t1) return;
    const bool partial = kt.n > a.split_tiles;

    const int r = tid >> 2, c = tid & 3, rr = rr0 + r, tok = head_group(a, rr), h = kvh * a.G + rr - tok * a.G;
    const bool live = rr < n_rows;
    const long long row = sq.row0 + tok;
    const int pos = live ? sq.past + tok : -1;
    const T* kc = static_cast<const T*>(p.cache.k) + kvh * p.cache.head_stride;
    const T* vc = static_cast<const T*>(p.cache.v) + kvh * p.cache.head_stride;
    auto load = [&](int t, int buf) {
        int start, end;
        key_range(kt, t, kSKeys, start, end);
        const long long off = start + r < end ? key_offset(p, s, start + r) : -1;
        if (c == 0) there[buf][r] = off >= 0;
        if (off < 0) return;  // (left as it is: nothing of it is used)
        float* kd = kv + (2 * buf * kSKeys + r) * ld;
        float* vd = kd + kSKeys * ld;
        if constexpr (sizeof(T) == 4) {
            const uint32_t ks = smem_u32(kd), vs = smem_u32(vd);
            if (vec) {
                for (int d = 4 * c; d < D; d += 16) {
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(ks + d * 4), "l"(kc + off + d) : "memory");
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(vs + d * 4), "l"(vc + off + d) : "memory");
                }
            } else {
                for (int d = c; d < D; d += 4) {
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(ks + d * 4), "l"(kc + off + d) : "memory");
                    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(vs + d * 4), "l"(vc + off + d) : "memory");
                }
            }
        } else {
            for (int d = c; d < D; d += 4) {
                kd[d] = to_f(kc[off + d]);
                vd[d] = to_f(vc[off + d]);
            }
        }
    };
    // the channels between D and D4 are zeros throughout
    if (D4 != D) {
        for (int i = tid; i < (kSRows + 4 * kSKeys) * 4; i += kSThreads)
            if (D + (i & 3) < D4) sm[(i >> 2) * ld + D + (i & 3)] = 0.f;
    }
    load(t0, 0);
    cp_async_commit();
    {
        const T* q = static_cast<const T*>(p.q) + row * p.ldq + static_cast<long long>(h) * D;
        for (int d = c; d < D; d += 4) Qs[r * ld + d] = live ? to_f(q[d]) : 0.f;
    }
    float4 o[DM / 16];
#pragma unroll
    for (int i = 0; i < DM / 16; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    float m = kNegInf, l = 0.f;

    for (int t = t0; t < t1; ++t) {
        const int buf = (t - t0) & 1;
        if (t + 1 < t1) load(t + 1, buf ^ 1);
        cp_async_commit();
        cp_async_wait<1>();
        __syncthreads();
        int start, end;
        key_range(kt, t, kSKeys, start, end);
        const float* Ks = kv + 2 * buf * kSKeys * ld;
        const float* Vs = Ks + kSKeys * ld;
        float sc[8] = {};
        const float4* qv = reinterpret_cast<const float4*>(Qs + r * ld);
#pragma unroll 2
        for (int d = 0; d < D4 / 4; ++d) {
            const float4 x = qv[d];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float4 y = *reinterpret_cast<const float4*>(Ks + (c + 4 * i) * ld + 4 * d);
                sc[i] = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, sc[i]))));
            }
        }
        float mx = kNegInf;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int key = c + 4 * i;
            float v = sc[i] * p.scale;
            if (p.softcap > 0.f) v = p.softcap * tanhf(v / p.softcap);
            sc[i] = there[buf][key] && seen(start + key, pos, p.window, p.sinks) ? v : kNegInf;
            mx = fmaxf(mx, sc[i]);
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float m_new = fmaxf(m, mx), base = m_new == kNegInf ? 0.f : m_new;
        const float alpha = ex2_approx((m - base) * kLog2e);
        m = m_new;
        l *= alpha;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            sc[i] = ex2_approx((sc[i] - base) * kLog2e);
            l += sc[i];
        }
#pragma unroll
        for (int i = 0; i < DM / 16; ++i) {
            o[i].x *= alpha, o[i].y *= alpha, o[i].z *= alpha, o[i].w *= alpha;
        }
        // a key that a row does not see has p = 0, and 0 * v is left out where v may not be finite for it
        const bool whole = end - start == kSKeys && all_seen(kt, start, end, p.window, p.sinks) &&
                           __all_sync(0xffffffffu, there[buf][tid & 31]);
        const int quad = tid & 28;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
#pragma unroll
            for (int cc = 0; cc < 4; ++cc) {
                const float pr = __shfl_sync(0xffffffffu, sc[i], quad | cc);
                if (!whole && pr == 0.f) continue;
                const float* v = Vs + (cc + 4 * i) * ld + 4 * c;
#pragma unroll
                for (int d = 0; d < DM / 16; ++d) {
                    if (4 * c + 16 * d < D4) {
                        const float4 y = *reinterpret_cast<const float4*>(v + 16 * d);
                        o[d].x = fmaf(pr, y.x, o[d].x);
                        o[d].y = fmaf(pr, y.y, o[d].y);
                        o[d].z = fmaf(pr, y.z, o[d].z);
                        o[d].w = fmaf(pr, y.w, o[d].w);
                    }
                }
            }
        }
        __syncthreads();  // before this tile's place is filled again
    }
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if (!live) return;
    const float inv = partial ? 1.f : (l > 0.f || l != l ? 1.f / l : 0.f);
    const long long at = (static_cast<long long>(split) * p.batch.rows + row) * p.q_heads + h;
    if (partial && c == 0) a.ml[at] = make_float2(m * kLog2e, l);  // base-2 exponents, as the other kernels'
    T* out = static_cast<T*>(p.out) + row * p.ldo + static_cast<long long>(h) * D;
#pragma unroll
    for (int i = 0; i < DM / 16; ++i) {
        const float v[4] = {o[i].x, o[i].y, o[i].z, o[i].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int d = 4 * c + 16 * i + e;
            if (d >= D) continue;
            if (partial) a.part[at * D + d] = v[e];
            else out[d] = from_f<T>(v[e] * inv);
        }
    }
}

// --- tensor cores, mma.sync -------------------------------------------------------------------
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf2(float lo, float hi) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&b);
}
// A pair of bf16 with what is not finite replaced by zero; `bad` is set where something was.
__device__ __forceinline__ uint32_t finite2(uint32_t x, bool& bad) {
    if ((x & 0x7f80u) == 0x7f80u) x &= 0xffff0000u, bad = true;
    if ((x & 0x7f800000u) == 0x7f800000u) x &= 0x0000ffffu, bad = true;
    return x;
}
// cap tanh(z) log2(e) of a product x, z = x scale / cap, for caps beyond kCheapCap (pattn.cuh has the cheap form, which
// cancels where |z| is small): below |z| = 1/4 the score itself times the Taylor series of tanh(z) / z up to z^8 (what
// follows is below 2^-26), from there on the cheap form, whose error is then 2^-19 of the score.
__device__ __forceinline__ float wide_cap_log2(float x, float to_z, float scale_log2, float cap_log2) {
    constexpr float kTwoLog2e = 2.885390081777927f;
    const float z = x * to_z, z2 = z * z;
    const float series = fmaf(z2, fmaf(z2, fmaf(z2, fmaf(z2, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
    return fabsf(z) < 0.25f ? x * scale_log2 * series : soft_cap_log2(z, kTwoLog2e, cap_log2);
}

// DP: padded head size. WIDE: soft caps beyond kCheapCap, a kernel of its own (as a branch, or for every cap, it cost
// single tokens at head size 256 3 %: 428 us for 64 behind 100 to 16000 tokens, 414 without). Groups of WM warps (16
// rows each) share out each step's 64 keys, 4 / WM groups: a single token's few rows keep all four
// warps busy on different keys. Every group runs on its own: it brings its keys and values into its
// own ring of ST tiles, waits for them alone (no block barrier in the loop), and every warp has its
// own softmax; the groups' results are joined once at the end. P is rounded to bf16 for the second
// product.
//
// Keys and values sit in slabs of 64 channels, rows of 128 bytes whose 16-byte chunks are swapped
// by the row number (c ^ (r & 7)), so that ldmatrix meets no bank twice. TMA: a page's keys come by
// one tensor copy per slab, which lays them out so. Otherwise (pages that end inside a group's
// keys) by 16-byte cp.async; the page lookups run a tile ahead of the loads.
// What bounds a decoding step is HBM, and short of it the latency of the loop's instructions.
template <int DP>
struct MmaShape {
    static constexpr int kKeys = 64;
    static constexpr int kStages = DP == 64 ? 4 : 3;
    static constexpr int kTileBytes = kKeys * DP * 2;
    // behind the tiles: the keys' offsets (cp.async; [kStages + 1][kKeys]) or the copies' barriers (TMA), and in the
    // end the statistics of up to 64 rows
    static __host__ __device__ constexpr int tail(bool tma) { return tma ? 512 + 4 * kStages * 8 : (kStages + 1) * kKeys * 8; }
    static __host__ __device__ constexpr int align(bool tma) { return tma ? 1024 : 128; }  // tensor copies: the swizzle's period
    static __host__ __device__ constexpr int smem(int rows, bool tma) {
        return align(tma) + rows * DP * 2 + kStages * 2 * kTileBytes + tail(tma);
    }
};

template <int DP, int WM, bool TMA, bool WIDE>
__global__ void __launch_bounds__(128) paged_mma_kernel(const __grid_constant__ Args a,
                                                        const __grid_constant__ CUtensorMap k_map,
                                                        const __grid_constant__ CUtensorMap v_map, const int box) {
    using Sh = MmaShape<DP>;
    constexpr int BN = Sh::kKeys, ST = Sh::kStages, BM = 16 * WM, WK = 4 / WM, GK = BN / WK, NT = GK / 8;
    extern __shared__ unsigned char smem_raw[];
    const PagedAttention& p = a.p;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wm = warp % WM, wk = warp / WM, D = p.cache.D;
    const int tile = a.row_tiles - 1 - static_cast<int>(blockIdx.x % a.row_tiles);
    const int rest = blockIdx.x / a.row_tiles, split = rest % a.splits, s = rest / a.splits, kvh = blockIdx.y;
    cudaTriggerProgrammaticLaunchCompletion();  // the join's blocks may take their places
    const Sequence sq = sequence(p, s, blockIdx.x % (a.row_tiles * a.splits) == 0 && kvh == 0 && tid == 0);
    const int rr0 = tile * BM, n_rows = sq.n_new * a.G;
    if (!sq.ok || rr0 >= n_rows) return;
    const KeyTiles kt = key_tiles(sq.past, sq.n_new, a.G, rr0, rr0 + BM, p.window, p.sinks, BN, a.align);
    const int t0 = split * a.split_tiles, n = min(kt.n, t0 + a.split_tiles) - t0;
    if (n <= 0) return;
    const bool partial = kt.n > a.split_tiles;

    constexpr uint32_t kAlign = Sh::align(TMA);
    const uint32_t q_s = (smem_u32(smem_raw) + kAlign - 1) & ~(kAlign - 1), kv_s = q_s + BM * DP * 2;
    unsigned char* smem = smem_raw + (q_s - smem_u32(smem_raw));
    constexpr int kOffs = BM * DP * 2 + ST * 2 * Sh::kTileBytes;
    // this group's part of all of it
    constexpr int kGroupTile = GK * DP * 2;
    const int gt = tid - wk * (32 * WM), kb = wk * GK;  // thread within the group; its first key of a tile
    const uint32_t ring = kv_s + wk * (ST * 2 * kGroupTile);
    long long* offs = reinterpret_cast<long long*>(smem + kOffs) + wk * (ST + 1) * GK;  // [ST + 1][GK], cp.async
    const uint32_t full = q_s + kOffs + 512 + wk * (ST * 8);                            // [ST] barriers, TMA
    auto group_all = [&](bool ok) -> bool {  // barrier of the group, with the conjunction of what its threads bring
        if (WM == 1) {
            const bool all_ok = __all_sync(0xffffffffu, ok);
            __syncwarp();  // a vote alone does not order the lanes' shared memory
            return all_ok;
        }
        int all;
        asm volatile(
            "{\n\t.reg .pred p, q;\n\tsetp.ne.s32 p, %1, 0;\n\tbar.red.and.pred q, %2, %3, p;\n\tselp.s32 %0, 1, 0, q;\n\t}"
            : "=r"(all)
            : "r"(ok ? 1 : 0), "r"(1 + wk), "n"(32 * WM)
            : "memory");
        return all != 0;
    };
    auto swz = [](int rows, int row, int chunk) {
        return static_cast<uint32_t>((chunk >> 3) * (rows * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
    };
    const int slabs = (D + 63) / 64;

    const bf16* q = static_cast<const bf16*>(p.q);
    for (int i = tid; i < BM * (DP / 8); i += 128) {
        const int r = i / (DP / 8), c = i % (DP / 8), rr = rr0 + r;
        const bool in = rr < n_rows && c * 8 < D;
        const int t = head_group(a, rr);
        const bf16* src = in ? q + (sq.row0 + t) * p.ldq + static_cast<long long>(kvh * a.G + rr - t * a.G) * D + c * 8 : q;
        cp_async16(q_s + swz(BM, r, c), src, in);
    }
    if (TMA) cp_async_commit();
    const bf16* kc = static_cast<const bf16*>(p.cache.k) + kvh * p.cache.head_stride;
    const bf16* vc = static_cast<const bf16*>(p.cache.v) + kvh * p.cache.head_stride;
    // cp.async: offset of this thread's key (gt < GK) of tile i
    auto offset_of = [&](int i) -> long long {
        int start, end;
        key_range(kt, t0 + i, BN, start, end);
        return start + kb + gt < end ? key_offset(p, s, start + kb + gt) : -1;
    };
    auto load = [&](int i) {
        const long long* of = offs + (i % (ST + 1)) * GK;
        const uint32_t ks = ring + (i % ST) * (2 * kGroupTile), vs = ks + kGroupTile;
        for (int slab = 0; slab < slabs; ++slab) {
            const int c = slab * 8 + (gt & 7);
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int key = x * (4 * WM) + (gt >> 3);
                const long long off = of[key];
                const bool in = off >= 0 && c * 8 < D;
                const long long e = in ? off + c * 8 : 0;
                cp_async16(ks + swz(GK, key, c), kc + e, in);
                cp_async16(vs + swz(GK, key, c), vc + e, in);
            }
        }
    };
    // TMA, the group's first warp: the page of this lane's box (lane < GK / box) of tile i, -1 for none; and the tile's copies
    auto page_of = [&](int i) -> int {
        int start, end;
        key_range(kt, t0 + i, BN, start, end);
        const int key = start + kb + lane * box;
        if (lane >= GK / box || key >= end) return -1;
        const int slot = page_slot(p, key);
        const int page = slot < p.batch.table_width ? p.batch.table[s * p.batch.table_stride + slot] : -1;
        return page < p.cache.pages ? page : -1;
    };
    auto copy = [&](int i, int page) {
        const uint32_t bar = full + 8u * (i % ST);
        const unsigned there = __ballot_sync(0xffffffffu, page >= 0);
        if (lane == 0) mbar_arrive_expect_tx(bar, static_cast<uint32_t>(__popc(there)) * box * 128 * 2 * slabs);
        __syncwarp();
        if (page < 0) return;
        int start, end;
        key_range(kt, t0 + i, BN, start, end);
        const int key = start + kb + lane * box, at = key - page_slot(p, key) * p.cache.page_size;
        const uint32_t ks = ring + (i % ST) * (2 * kGroupTile) + lane * box * 128;
        for (int slab = 0; slab < slabs; ++slab) {
            tma_load_4d(&k_map, ks + slab * (GK * 128), bar, slab * 64, at, kvh, page);
            tma_load_4d(&v_map, ks + kGroupTile + slab * (GK * 128), bar, slab * 64, at, kvh, page);
        }
    };
    bool bad_page = false;
    int next_page = -1;
    if (TMA) {
        if (tid == 0) {
            for (int i = 0; i < WK * ST; ++i) mbar_init(q_s + kOffs + 512 + 8u * i, 1);
            fence_barrier_init();
        }
        bad_page = __syncthreads_or(any_bad_page(p, s, kt, t0, n, BN));
        if (wm == 0) {
#pragma unroll
            for (int i = 0; i < ST - 1; ++i)
                if (i < n) copy(i, page_of(i));
            if (ST - 1 < n) next_page = page_of(ST - 1);
        }
        cp_async_wait<0>();
        __syncthreads();  // q is there
    } else {
        if (gt < GK) {
#pragma unroll
            for (int i = 0; i < ST; ++i) offs[i * GK + gt] = i < n ? offset_of(i) : -1;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < ST - 1; ++i) {
            if (i < n) load(i);
            cp_async_commit();
        }
        cp_async_wait<ST - 2>();
        __syncthreads();  // every thread's part of q (and of tile 0) is there
    }

    float o[DP / 8][4];
#pragma unroll
    for (int i = 0; i < DP / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    // The divisor is the sum of the rounded probabilities (the weights then sum to 1: see pattn_tc.cu), which one more
    // product with a matrix of ones gives, the same in every column.
    float m[2] = {kNegInf, kNegInf}, sums[4] = {0.f, 0.f, 0.f, 0.f};
    constexpr uint32_t kOnes = 0x3f803f80u;
    int pos[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int rr = rr0 + wm * 16 + (lane >> 2) + 8 * i;
        pos[i] = rr < n_rows ? sq.past + head_group(a, rr) : -1;
    }
    const float scale_log2 = p.scale * kLog2e;
    const float cap_in = p.softcap > 0.f ? (WIDE ? p.scale : 2.f * scale_log2) / p.softcap : 0.f, cap_out = p.softcap * kLog2e;

    // A lane's part of the ldmatrix addresses: its row, and its chunk of the first 16 channels of a slab, swapped by the
    // row; the other channels' chunks differ in bits 5 and 6 (^ 32 per 16 channels).
    const uint32_t q_lane = swz(BM, wm * 16 + (lane & 15), lane >> 4);
    const uint32_t k_lane = swz(GK, (lane & 7) + ((lane >> 4) << 3), (lane >> 3) & 1);
    const uint32_t v_lane = swz(GK, lane & 15, lane >> 4);
    constexpr bool kQRegs = DP <= 128;  // q's operands stay in registers
    uint32_t qf[kQRegs ? DP / 16 : 1][4];
    if constexpr (kQRegs) {
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) ldmatrix4(qf[kk], q_s + (kk >> 2) * (BM * 128) + (q_lane ^ ((kk & 3) << 5)));
    }

    for (int i = 0; i < n; ++i) {
        long long next = -1;
        if (TMA) {
            const bool ok = mbar_wait(full + 8u * (i % ST), (i / ST) & 1, p.err, kTimeout);
            if (!group_all(ok)) {  // the group leaves together; what is on its way lands first
                for (int x = i; x < min(n, i + ST - 1); ++x) mbar_wait_quiet(full + 8u * (x % ST), (x / ST) & 1);
                break;
            }
            if (wm == 0) {
                if (i + ST - 1 < n) copy(i + ST - 1, next_page);
                if (i + ST < n) next_page = page_of(i + ST);
            }
        } else {
            cp_async_wait<ST - 2>();
            group_all(true);
            if (i + ST - 1 < n) load(i + ST - 1);
            cp_async_commit();
            if (gt < GK && i + ST < n) next = offset_of(i + ST);
        }

        const uint32_t ks = ring + (i % ST) * (2 * kGroupTile), vs = ks + kGroupTile;
        // Scores; two chains of products per score where a warp has few scores.
        float sc[NT][4], sd[2][4];
#pragma unroll
        for (int t = 0; t < NT; ++t) sc[t][0] = sc[t][1] = sc[t][2] = sc[t][3] = 0.f;
#pragma unroll
        for (int t = 0; t < 2; ++t) sd[t][0] = sd[t][1] = sd[t][2] = sd[t][3] = 0.f;
#pragma unroll
        for (int kk = 0; kk < DP / 16; ++kk) {
            if (kk < 12 || slabs == 4) {  // channels of a slab behind D are zeros
                uint32_t qa[4];
                if constexpr (kQRegs) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) qa[x] = qf[kk][x];
                } else {
                    ldmatrix4(qa, q_s + (kk >> 2) * (BM * 128) + (q_lane ^ ((kk & 3) << 5)));
                }
#pragma unroll
                for (int t = 0; t < NT / 2; ++t) {
                    uint32_t b[4];
                    ldmatrix4(b, ks + (kk >> 2) * (GK * 128) + t * 2048 + (k_lane ^ ((kk & 3) << 5)));
                    if (NT == 2 && (kk & 1)) {
                        mma16816(sd[0], qa, b[0], b[1]);
                        mma16816(sd[1], qa, b[2], b[3]);
                    } else {
                        mma16816(sc[2 * t], qa, b[0], b[1]);
                        mma16816(sc[2 * t + 1], qa, b[2], b[3]);
                    }
                }
            }
        }
        if (NT == 2) {
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[0][e] += sd[0][e], sc[1][e] += sd[1][e];
        }
        int start, end;
        key_range(kt, t0 + i, BN, start, end);
        start += kb;  // of the group
        const long long* of = offs + (i % (ST + 1)) * GK;
        auto there = [&](int key) {  // key of the tile exists: it is in the range and its page in the pool
            return TMA ? start + key < end && (!bad_page || key_offset(p, s, start + key) >= 0) : of[key] >= 0;
        };
        const bool missing = TMA ? end - start < GK || bad_page
                                 : __any_sync(0xffffffffu, of[lane % GK] < 0 || (GK == 64 && of[(lane + 32) % GK] < 0));
        const bool whole = !missing && all_seen(kt, start, min(end, start + GK), p.window, p.sinks);
        if (p.softcap > 0.f) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    sc[t][e] = WIDE ? wide_cap_log2(sc[t][e], cap_in, scale_log2, cap_out) : soft_cap_log2(sc[t][e], cap_in, cap_out);
        } else {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[t][e] *= scale_log2;
        }
        if (!whole) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int key = t * 8 + (lane & 3) * 2 + (e & 1);
                    if (!there(key) || !seen(start + key, pos[e >> 1], p.window, p.sinks)) sc[t][e] = kNegInf;
                }
        }
        // The rows' maxima are shared out among lanes only where a lane has a score above its row's, which is seldom after
        // the first tiles (the largest probability is then exactly 1, and its rounding exact).
        float mx[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            mx[r] = fmaxf(sc[0][2 * r], sc[0][2 * r + 1]);
#pragma unroll
            for (int t = 1; t < NT; ++t) mx[r] = fmaxf(mx[r], fmaxf(sc[t][2 * r], sc[t][2 * r + 1]));
        }
        if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1])) {
            float alpha[2];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 1));
                mx[r] = fmaxf(mx[r], __shfl_xor_sync(0xffffffffu, mx[r], 2));
                const bool move = mx[r] > m[r];
                alpha[r] = move ? ex2_approx(m[r] - mx[r]) : 1.f;
                m[r] = move ? mx[r] : m[r];
                sums[2 * r] *= alpha[r], sums[2 * r + 1] *= alpha[r];
            }
#pragma unroll
            for (int d = 0; d < DP / 8; ++d) {
                o[d][0] *= alpha[0], o[d][1] *= alpha[0];
                o[d][2] *= alpha[1], o[d][3] *= alpha[1];
            }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const float base = m[r] == kNegInf ? 0.f : m[r];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                sc[t][2 * r] = ex2_approx(sc[t][2 * r] - base);
                sc[t][2 * r + 1] = ex2_approx(sc[t][2 * r + 1] - base);
            }
        }
        bool bad = false;
        auto values = [&](auto clean) {
#pragma unroll
            for (int t = 0; t < NT / 2; ++t) {
                const uint32_t pa[4] = {pack_bf2(sc[2 * t][0], sc[2 * t][1]), pack_bf2(sc[2 * t][2], sc[2 * t][3]),
                                        pack_bf2(sc[2 * t + 1][0], sc[2 * t + 1][1]),
                                        pack_bf2(sc[2 * t + 1][2], sc[2 * t + 1][3])};
                mma16816(sums, pa, kOnes, kOnes);
#pragma unroll
                for (int d = 0; d < DP / 16; ++d) {
                    if (d < 12 || slabs == 4) {
                        uint32_t b[4];
                        ldmatrix4_t(b, vs + (d >> 2) * (GK * 128) + t * 2048 + (v_lane ^ ((d & 3) << 5)));
                        if constexpr (decltype(clean)::value) {  // 0 * v must be 0 for the rows that do not see v
#pragma unroll
                            for (int x = 0; x < 4; ++x) b[x] = finite2(b[x], bad);
                        }
                        mma16816(o[2 * d], pa, b[0], b[1]);
                        mma16816(o[2 * d + 1], pa, b[2], b[3]);
                    }
                }
            }
        };
        if (whole) values(std::false_type{});
        else values(std::true_type{});
        if (!whole && __any_sync(0xffffffffu, bad)) {
            // what finite2 took out, given back to the rows that see it
            for (int key = 0; key < GK; ++key) {
                if (!there(key)) continue;
                const bool s0 = seen(start + key, pos[0], p.window, p.sinks);
                const bool s1 = seen(start + key, pos[1], p.window, p.sinks);
                const unsigned char* vrow = smem + (vs - q_s);
#pragma unroll
                for (int d = 0; d < DP / 8; ++d) {
                    const uint32_t x = *reinterpret_cast<const uint32_t*>(vrow + swz(GK, key, d) + (lane & 3) * 4);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float v = __uint_as_float(e ? x & 0xffff0000u : x << 16);
                        if ((__float_as_uint(v) & 0x7f800000u) != 0x7f800000u) continue;
                        if (s0) o[d][e] += v;
                        if (s1) o[d][2 + e] += v;
                    }
                }
            }
        }
        if (!TMA && gt < GK) offs[((i + ST) % (ST + 1)) * GK + gt] = next;
    }
    cp_async_wait<0>();
    __syncthreads();
    // [WK][BM] rows of DP fp32 over the tiles' memory, and (max, sum) behind it
    constexpr int LD = DP + 8;
    static_assert(WK * BM * LD * 4 <= ST * 2 * Sh::kTileBytes, "the join fits the tiles' memory");
    static_assert(WK * BM * 8 <= 512, "the statistics fit the memory behind the tiles");
    float* os = reinterpret_cast<float*>(smem + BM * DP * 2);
    float2* st = reinterpret_cast<float2*>(smem + kOffs);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int row = wk * BM + wm * 16 + (lane >> 2) + 8 * r;
        if ((lane & 3) == 0) st[row] = make_float2(m[r], sums[2 * r]);
#pragma unroll
        for (int d = 0; d < DP / 8; ++d)
            *reinterpret_cast<float2*>(os + row * LD + d * 8 + (lane & 3) * 2) = make_float2(o[d][2 * r], o[d][2 * r + 1]);
    }
    __syncthreads();
    const int d8 = D / 8;
    for (int i = tid; i < BM * d8; i += 128) {
        const int r = i / d8, d = (i - r * d8) * 8, rr = rr0 + r;
        if (rr >= n_rows) break;
        float mm = kNegInf, ll = 0.f, v[8] = {};
#pragma unroll
        for (int w = 0; w < WK; ++w) mm = fmaxf(mm, st[w * BM + r].x);
        const float base = mm == kNegInf ? 0.f : mm;
#pragma unroll
        for (int w = 0; w < WK; ++w) {
            const float2 x = st[w * BM + r];
            const float f = ex2_approx(x.x - base);
            ll = fmaf(x.y, f, ll);
            const float* src = os + (w * BM + r) * LD + d;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = fmaf(src[e], f, v[e]);
        }
        const int t = head_group(a, rr), h = kvh * a.G + rr - t * a.G;
        const long long row = sq.row0 + t;
        if (partial) {
            const long long at = (static_cast<long long>(split) * p.batch.rows + row) * p.q_heads + h;
            if (d == 0) a.ml[at] = make_float2(mm, ll);
            float4* dst = reinterpret_cast<float4*>(a.part + at * D + d);
            dst[0] = make_float4(v[0], v[1], v[2], v[3]);
            dst[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            const float inv = ll == 0.f ? 0.f : 1.f / ll;
            *reinterpret_cast<uint4*>(static_cast<bf16*>(p.out) + row * p.ldo + static_cast<long long>(h) * D + d) =
                make_uint4(pack_bf2(v[0] * inv, v[1] * inv), pack_bf2(v[2] * inv, v[3] * inv),
                           pack_bf2(v[4] * inv, v[5] * inv), pack_bf2(v[6] * inv, v[7] * inv));
        }
    }
}

// --- joining the splits -----------------------------------------------------------------------
// One block per row and head. The splits' maxima give their weights (shared memory, kSome at a time);
// the warps share out the splits, and each lane sums its channels over its warp's, then over the warps
// in order. It is launched beside the kernel before it and waits for that one's end on the device, so
// that its own start is not added to a decoding step.
constexpr int kSome = 128;
template <class T>
__global__ void __launch_bounds__(128) paged_combine_kernel(const __grid_constant__ Args a) {
    __shared__ float weight[kSome];
    __shared__ float red[4];
    __shared__ float sums[4][256];
    const PagedAttention& p = a.p;
    const int row = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, D = p.cache.D;
    int s = 0;
    for (int s0 = 0; s0 < p.batch.S; s0 += 128) {
        const int i = s0 + tid;
        s += __syncthreads_count(i < p.batch.S && p.batch.row_start[i + 1] <= row);
    }
    int active = 0;
    if (s < p.batch.S) {
        const Sequence sq = sequence(p, s, false);
        if (sq.ok && row >= sq.row0 && row - sq.row0 < sq.n_new) {
            const int rr = (row - sq.row0) * a.G + h % a.G, tile = rr / a.BM;
            const KeyTiles kt = key_tiles(sq.past, sq.n_new, a.G, tile * a.BM, (tile + 1) * a.BM, p.window, p.sinks, a.BN, a.align);
            active = (kt.n + a.split_tiles - 1) / a.split_tiles;
        }
    }
    cudaGridDependencySynchronize();
    if (active <= 1) return;  // written already, or not to be written
    const long long step = static_cast<long long>(p.batch.rows) * p.q_heads;
    const long long at = static_cast<long long>(row) * p.q_heads + h;
    float m = kNegInf;
    for (int i = tid; i < active; i += 128) m = fmaxf(m, a.ml[at + i * step].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) red[warp] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float base = m == kNegInf ? 0.f : m;
    float acc[8] = {}, l = 0.f;
    for (int i0 = 0; i0 < active; i0 += kSome) {
        __syncthreads();
        if (i0 + tid < active) {
            const float2 x = a.ml[at + (i0 + tid) * step];
            const float f = ex2_approx(x.x - base);
            weight[tid] = f;
            l = fmaf(x.y, f, l);
        }
        __syncthreads();
        const int n = min(kSome, active - i0);
#pragma unroll 4
        for (int i = warp; i < n; i += 4) {
            const float f = weight[i];
            const float* src = a.part + (at + (i0 + i) * step) * D;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (lane + 32 * e < D) acc[e] = fmaf(src[lane + 32 * e], f, acc[e]);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
    __syncthreads();
    if (lane == 0) red[warp] = l;
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[warp][lane + 32 * e] = acc[e];
    __syncthreads();
    l = (red[0] + red[1]) + (red[2] + red[3]);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    T* out = static_cast<T*>(p.out) + static_cast<long long>(row) * p.ldo + static_cast<long long>(h) * D;
    for (int d = tid; d < D; d += 128)
        out[d] = from_f<T>(((sums[0][d] + sums[1][d]) + (sums[2][d] + sums[3][d])) * inv);
}

// --- plan and launch ----------------------------------------------------------------------------
enum Kind { kSimt, kMma, kTc };

// The tcgen05 kernel's 128-row tiles take over from the mma.sync kernel above so many packed rows of the longest chunk.
// Measured on 1, 16 and 64 sequences behind 8000, 2000 and 300 tokens, us with mma.sync / with tcgen05: head size 64, 48 and
// 128 rows, 29.5 / 30.9 and 57.7 / 43.5 (16 sequences); 128, 32 and 48 rows, 28.7 / 33.0 and 57.4 / 35.1; 256, 8 and 18 rows,
// 41.2 / 40.6 and 53.5 / 37.9.
bool wants_tc(const PagedAttention& p) {
    const int rows = p.cache.D <= 64 ? 64 : p.cache.D <= 128 ? 32 : 16;
    return static_cast<long long>(p.batch.max_new) * (p.q_heads / p.cache.kv_heads) > rows;
}

bool cache_fits_mma(const PagedCache& c) {
    return c.dtype == kBf16 && c.D % 8 == 0 && (reinterpret_cast<uintptr_t>(c.k) & 15) == 0 &&
           (reinterpret_cast<uintptr_t>(c.v) & 15) == 0 && c.page_stride % 8 == 0 && c.token_stride % 8 == 0 &&
           c.head_stride % 8 == 0;
}

// The launch of one kind: tiles and splits, by sizes that the host knows.
Args plan(const PagedAttention& p, Kind kind, int num_sms) {
    Args a{};
    a.p = p;
    a.G = p.q_heads / p.cache.kv_heads;
    a.g_div = page_divisor(a.G);
    const long long packed = static_cast<long long>(p.batch.max_new) * a.G;
    a.align = 1;
    int resident;  // blocks per SM
    if (kind == kSimt) {
        a.BM = kSRows;
        a.BN = kSKeys;
        resident = 2;
    } else if (kind == kTc) {
        a.BM = tc_rows(p.cache.D);
        a.BN = tc_keys();
        a.align = std::max(1, copy_box(p.cache, a.BN));
        resident = 1;
    } else {
        a.BM = packed <= 16 ? 16 : packed <= 32 ? 32 : 64;
        a.BN = 64;
        a.align = std::max(1, copy_box(p.cache, a.BM));  // a group brings as many keys as a block has rows
        resident = p.cache.D > 128 ? 1 : 2;
    }
    a.row_tiles = std::max(1, ceil_div(packed, a.BM));  // (max_new 0: the checks still run)
    const long long span = p.window > 0 ? std::min<long long>(p.batch.max_kv, static_cast<long long>(p.window) + p.batch.max_new +
                                                                                 p.sinks)
                                        : p.batch.max_kv;
    // a window's sinks and its start, rounded down to `align`, may each take part of one tile more
    const int tiles = ceil_div(span, a.BN) + (p.window > 0 ? (a.align > 1 ? 2 : 1) : 0);
    const long long base = static_cast<long long>(p.batch.S) * p.cache.kv_heads * a.row_tiles;
    // Splits fill one wave, in shares of three tiles or more (one sequence of 2000 tokens, 8 heads of 128 over 4: 12.4 us;
    // shares of eight tiles 16.5; of two no less, while a short cache then pays for the join). Beyond one wave, sequences
    // of different lengths, of which only the longest is known here, even out in blocks of a sixteenth of a wave's share (64
    // sequences of 100 to 16000 tokens: 4, 8, 16 and 32 waves 314, 299, 305 and 340 us), but in shares of eight tiles: 64
    // sequences of 1500 tokens took 48 us so, and 56 in shares of three. The CUDA-core kernel's tiles take longer.
    const long long slots = static_cast<long long>(num_sms) * resident, per = std::max<long long>(base, 1);
    long long splits = slots / per;
    if (kind == kMma && p.batch.S > 1) splits = std::max<long long>(splits, std::min<long long>(16 * slots / per, tiles / 8));
    if (kind == kSimt && p.batch.S > 1) splits = 4 * slots / per;
    splits = std::max<long long>(1, std::min<long long>(splits, tiles / (kind == kSimt ? 2 : 3)));
    a.split_tiles = std::max(1, ceil_div(tiles, splits));
    a.splits = std::max(1, ceil_div(tiles, a.split_tiles));  // (max_kv 0: the checks still run)
    return a;
}

size_t part_bytes(const Args& a) {
    if (a.splits <= 1) return 0;
    const size_t n = static_cast<size_t>(a.splits) * a.p.batch.rows * a.p.q_heads;
    const size_t ml = (n * sizeof(float2) + 15) & ~static_cast<size_t>(15);
    return ml + n * a.p.cache.D * sizeof(float);
}

void raise_smem(const void* f, int bytes, PerDeviceOnce& once) {
    if (!once.pending()) return;
    SANA_CUDA(cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    once.mark();
}

template <int DP, int WM, bool TMA, bool WIDE>
void launch_mma(const Args& a, int box, dim3 grid, cudaStream_t st) {
    static PerDeviceOnce once;
    constexpr int bytes = MmaShape<DP>::smem(16 * WM, TMA);
    static_assert(bytes <= 232448, "shared memory of one block");
    raise_smem(reinterpret_cast<const void*>(&paged_mma_kernel<DP, WM, TMA, WIDE>), bytes, once);
    CUtensorMap k{}, v{};
    if (TMA) {
        k = pool_map(a.p.cache, a.p.cache.k, box);
        v = pool_map(a.p.cache, a.p.cache.v, box);
    }
    paged_mma_kernel<DP, WM, TMA, WIDE><<<grid, 128, bytes, st>>>(a, k, v, box);
}

template <int DP, int WM>
void launch_mma(const Args& a, dim3 grid, cudaStream_t st) {
    const int box = copy_box(a.p.cache, 16 * WM);  // within a group's keys
    const bool wide = a.p.softcap > kCheapCap;
    if (box > 0) wide ? launch_mma<DP, WM, true, true>(a, box, grid, st) : launch_mma<DP, WM, true, false>(a, box, grid, st);
    else wide ? launch_mma<DP, WM, false, true>(a, 0, grid, st) : launch_mma<DP, WM, false, false>(a, 0, grid, st);
}

template <int DP>
void launch_mma_rows(const Args& a, dim3 grid, cudaStream_t st) {
    if (a.BM == 16) launch_mma<DP, 1>(a, grid, st);
    else if (a.BM == 32) launch_mma<DP, 2>(a, grid, st);
    else launch_mma<DP, 4>(a, grid, st);
}

template <class T, int DM>
void launch_simt(const Args& a, dim3 grid, cudaStream_t st) {
    static PerDeviceOnce once;
    constexpr int most = (kSRows + 4 * kSKeys) * (DM + 4) * 4;
    static_assert(most <= 232448, "shared memory of one block");
    raise_smem(reinterpret_cast<const void*>(&paged_simt_kernel<T, DM>), most, once);
    const PagedCache& c = a.p.cache;
    const int ld = ((c.D + 3) & ~3) + 4;
    const bool vec = c.D % 4 == 0 && c.page_stride % 4 == 0 && c.token_stride % 4 == 0 && c.head_stride % 4 == 0 &&
                     (reinterpret_cast<uintptr_t>(c.k) & 15) == 0 && (reinterpret_cast<uintptr_t>(c.v) & 15) == 0;
    paged_simt_kernel<T, DM><<<grid, kSThreads, (kSRows + 4 * kSKeys) * ld * 4, st>>>(a, vec ? 1 : 0);
}
template <class T>
void launch_simt(const Args& a, dim3 grid, cudaStream_t st) {
    if (a.p.cache.D <= 64) launch_simt<T, 64>(a, grid, st);
    else if (a.p.cache.D <= 128) launch_simt<T, 128>(a, grid, st);
    else launch_simt<T, 256>(a, grid, st);
}

}  // namespace

// With l = ceil(log2 d): x / d = (mulhi(x, 2^(32+l) / d - 2^32 + 1) + x) >> l for x < 2^31 / 2 and any d >= 1, since the
// magic number exceeds 2^32 (2^l / d - 1) by at most 1 and x / 2^32 < 1 / (2 d) of a step is left.
PageDivisor page_divisor(int d) {
    PageDivisor v{0, 0};
    while ((1LL << v.shift) < d) ++v.shift;
    v.magic = static_cast<uint32_t>(((1ULL << 32) * ((1ULL << v.shift) - static_cast<unsigned>(d))) / static_cast<unsigned>(d) + 1);
    return v;
}

// Boxes are whole groups of eight rows, which the swizzle needs. A tensor map's strides end at 2^40 bytes; a stride of 0
// (other than of a size 1) is not encoded.
int copy_box(const PagedCache& c, int keys) {
    const long long most = 1LL << 38;
    const bool strides_ok = c.page_stride < most && c.token_stride < most && c.head_stride < most &&
                            (c.page_stride >= 8 || c.pages == 1) && (c.token_stride >= 8 || c.page_size == 1) &&
                            (c.head_stride >= 8 || c.kv_heads == 1);
    if (!strides_ok || c.pages < 1) return 0;
    if (c.page_size % keys == 0) return keys;
    return c.page_size % 8 == 0 && keys % c.page_size == 0 ? c.page_size : 0;
}

namespace {
cuuint64_t map_stride(long long elements) { return static_cast<cuuint64_t>(elements > 8 ? elements * 2 : 16); }
}  // namespace
CUtensorMap pool_map_slabs(const PagedCache& c, const void* base, int box) {
    CUtensorMap m;
    const cuuint64_t dims[5] = {64, static_cast<cuuint64_t>(c.page_size), static_cast<cuuint64_t>(c.D / 64),
                                static_cast<cuuint64_t>(c.kv_heads), static_cast<cuuint64_t>(c.pages)};
    const cuuint64_t strides[4] = {map_stride(c.token_stride), 128, map_stride(c.head_stride), map_stride(c.page_stride)};
    const cuuint32_t b[5] = {64, static_cast<cuuint32_t>(box), static_cast<cuuint32_t>(c.D / 64), 1, 1};
    tma_encode_tiled(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, base, dims, strides, b, CU_TENSOR_MAP_SWIZZLE_128B);
    return m;
}
CUtensorMap pool_map(const PagedCache& c, const void* base, int box) {
    CUtensorMap m;
    auto stride = map_stride;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(c.D), static_cast<cuuint64_t>(c.page_size),
                                static_cast<cuuint64_t>(c.kv_heads), static_cast<cuuint64_t>(c.pages)};
    const cuuint64_t strides[3] = {stride(c.token_stride), stride(c.head_stride), stride(c.page_stride)};
    const cuuint32_t b[4] = {64, static_cast<cuuint32_t>(box), 1, 1};
    tma_encode_tiled(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, base, dims, strides, b, CU_TENSOR_MAP_SWIZZLE_128B);
    return m;
}
}  // namespace pattn

using namespace pattn;

// Alignment of q and out, and the scale, are not known when the workspace is asked for: the largest of the kinds' needs.
size_t paged_attention_workspace(const PagedAttention& p, int num_sms) {
    size_t n = part_bytes(plan(p, kSimt, num_sms));
    if (cache_fits_mma(p.cache)) {
        n = std::max(n, part_bytes(plan(p, kMma, num_sms)));
        if (wants_tc(p)) n = std::max(n, part_bytes(plan(p, kTc, num_sms)));
    }
    return n;
}

void paged_attention(PagedAttention p, int num_sms, cudaStream_t st) {
    p.page_div = page_divisor(p.cache.page_size);
    if (p.batch.S == 0 || p.batch.rows == 0) return;
    const bool mma = cache_fits_mma(p.cache) && (reinterpret_cast<uintptr_t>(p.q) & 15) == 0 &&
                     (reinterpret_cast<uintptr_t>(p.out) & 15) == 0 && p.ldq % 8 == 0 && p.ldo % 8 == 0;
    // the tcgen05 kernel maps a tile's largest score alone, which takes a map that rises: scale > 0; and it has the cheap
    // form of the soft cap only (2048 tokens after 8192, head size 128: 646 us there, 1992 with the other form here)
    const Kind kind = !mma ? kSimt : wants_tc(p) && p.scale > 0.f && p.softcap <= kCheapCap ? kTc : kMma;
    Args a = plan(p, kind, num_sms);
    const size_t n = static_cast<size_t>(a.splits) * p.batch.rows * p.q_heads;
    a.ml = static_cast<float2*>(p.workspace);
    a.part = reinterpret_cast<float*>(static_cast<char*>(p.workspace) + ((n * sizeof(float2) + 15) & ~static_cast<size_t>(15)));
    const long long blocks = static_cast<long long>(p.batch.S) * a.splits * a.row_tiles;
    SANA_REQUIRE(blocks <= 0x7fffffffLL, "paged attention: too many sequences times row tiles for one launch");
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(p.cache.kv_heads));
    if (kind == kTc) {
        launch_tc(a, grid, st);
    } else if (mma) {
        if (p.cache.D <= 64) launch_mma_rows<64>(a, grid, st);
        else if (p.cache.D <= 128) launch_mma_rows<128>(a, grid, st);
        else launch_mma_rows<256>(a, grid, st);
    } else if (p.cache.dtype == kF32) {
        launch_simt<float>(a, grid, st);
    } else {
        launch_simt<bf16>(a, grid, st);
    }
    SANA_CUDA(cudaGetLastError());
    if (a.splits > 1) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(static_cast<unsigned>(p.batch.rows), static_cast<unsigned>(p.q_heads));
        cfg.blockDim = dim3(128);
        cfg.stream = st;
        cudaLaunchAttribute early{};
        early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        early.val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = &early;
        cfg.numAttrs = 1;
        if (p.cache.dtype == kF32) SANA_CUDA(cudaLaunchKernelEx(&cfg, paged_combine_kernel<float>, a));
        else SANA_CUDA(cudaLaunchKernelEx(&cfg, paged_combine_kernel<bf16>, a));
        SANA_CUDA(cudaGetLastError());
    }
}

}  // namespace sana
