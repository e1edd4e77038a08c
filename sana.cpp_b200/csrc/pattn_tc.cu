// Attention of a chunk of new tokens over a paged cache on the 5th-generation tensor cores
// (tcgen05), for chunks whose packed rows fill 128-row tiles; pattn.cuh has the packing, key
// ranges and splits, pattn.cu the other kernels and the choice between them.
//
// One block holds 256 packed rows as two tiles of 128 (one tile for head sizes above 128, whose
// output fills the tensor memory, and where fewer rows are left) and walks the key tiles of 128:
//   S = Q K^T into tensor memory; a thread per row reads its scores, masks them where the tile is
//   not seen whole, and writes P = 2^(s - m) as bf16 over S; O += P V with P from tensor memory.
// S has two slots. With two row tiles each has its own; with one, key tiles take them in turn. The
// issuing warp runs S(0), S(1), then PV(u), S(u + 2) for every S tile u, so that the tensor cores
// have the other slot's products while the softmax of one is under way, and S(u + 2) may overwrite
// P(u) since products run in order. (Two threads per row, or an issuing warp per slot, let both
// slots fall into step, all products waiting for all softmaxes: 277 us where this took 186.)
//
// The running maximum is a reference that moves only when a row's maximum passes it by 8 (a
// factor of 256): the output is rescaled in tensor memory then, by the row's own threads, and
// almost never after the first tiles. P stays below 2^8, its rounding to bf16 is relative, and the
// division at the end takes the reference out. The divisor is the fp32 sum of the rounded P, so that
// the weights still sum to 1: with a reference that is not the maximum the largest weights are
// rounded too, and the sum of the unrounded ones leaves an error 1.4 times that of the output's own
// rounding (1.05 to 1.4 times now, the less the fewer keys count), for 3 % of the time at head size
// 128. At 64, where all hangs on the softmax, it would be 17 %: there the sum is of the unrounded P.
//
// Keys and values come into the 128-byte-swizzled layout of the matrix descriptors: slabs of 64
// channels, 128-byte rows, chunk c of row r at c ^ (r & 7); K and Q are K-major operands, V is
// MN-major (its channels contiguous). K and V have a ring each, filled by warps of their own, of
// whole tiles, or for head sizes above 128, where a tile has 64 KB, of quarters (64 channels of K,
// 32 keys of V). Where pages divide a tile or tiles divide a page, tensor copies (TMA) bring them:
// one per page and slab. Above 128, V's keys stand in blocks of a product's 16 (8 where pages are of
// 8), [block][slab][key], which makes a copy of all slabs one box where the head size is a multiple of 64.
// Other page sizes end anywhere inside a tile and come by 16-byte cp.async.
#include <type_traits>

#include "pattn.cuh"
#include "tcgen05.cuh"
#include "tma.h"

namespace sana {
namespace pattn {
namespace {

using namespace tc;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kSoftmaxWarps = 8, kKeyWarp = 8, kValueWarp = 9, kMmaWarp = 11;  // (two value warps)
constexpr int kThreads = 12 * 32;
constexpr int kValueThreads = 64;
constexpr int kKeys = 128;  // per key tile

template <int DP>
struct TcShape {
    static constexpr int kTiles = DP <= 128 ? 2 : 1;     // row tiles of 128
    static constexpr int kRows = 128 * kTiles;
    static constexpr int kParts = kTiles == 2 ? 1 : 2;   // threads of a row
    static constexpr int kCols = kKeys / kParts;         // scores of a thread
    static constexpr int kSlabs = DP / 64;
    static constexpr int kPieces = DP <= 128 ? 1 : 4;    // of a tile of K or V
    static constexpr int kPieceSlabs = kSlabs / kPieces; // of K
    static constexpr int kPieceKeys = kKeys / kPieces;   // of V
    static constexpr int kBlock = DP <= 128 ? kKeys : 16;  // keys of a block of V (8 of them where pages are of 8)
    static constexpr int kPieceBytes = kKeys * DP * 2 / kPieces;
    static constexpr int kKRing = DP == 64 ? 4 : DP == 128 ? 2 : 4, kVRing = DP == 64 ? 4 : DP == 128 ? 2 : 5;  // pieces
    static constexpr int kQBytes = kTiles * 128 * DP * 2;
    static constexpr int kBarriers = 2 * (kKRing + kVRing) + 8 + 3;
    // behind Q and the rings: keys' offsets [2 for K, 2 for V][kKeys] (cp.async), maxima [2][kParts][128], barriers, three words
    static constexpr int kVRingAt = kQBytes + kKRing * kPieceBytes;
    static constexpr int kOffs = kVRingAt + kVRing * kPieceBytes;
    static constexpr int kMax = kOffs + 4 * kKeys * 8;
    static constexpr int kBars = kMax + (kParts > 1 ? 2 * kParts * 128 * 4 : 0);
    static constexpr int kSmem = 1024 + kBars + kBarriers * 8 + 16;
    // tensor memory columns: S slots at 0 and kKeys, O behind them
    static constexpr int kO = 2 * kKeys;
    static_assert(kO + kTiles * DP <= 512, "tensor memory");
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool in) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// The products and commits of the issuing warp, by the lane whose `on` is not 0: predicated, not branched around, so that
// the descriptors' arithmetic stays uniform. D += A B with A in shared memory, or (bf16 pairs) in tensor memory.
__device__ __forceinline__ void umma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate,
                                        uint32_t on) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(on)
        : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate,
                                        uint32_t on) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(on)
        : "memory");
}
__device__ __forceinline__ void umma_commit_on(uint32_t bar, uint32_t on) {
    asm volatile(
        "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
        "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(on)
        : "memory");
}
// Descriptor of an MN-major operand in the 128-byte swizzle: 64 channels of a row contiguous, groups
// of eight rows `group` bytes apart (the stride offset), slabs of 64 channels `slab` bytes apart (the
// leading offset).
__device__ __forceinline__ uint64_t mnmajor_sw128_desc(uint32_t smem_addr, uint32_t slab, uint32_t group) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu);
    d |= static_cast<uint64_t>((slab >> 4) & 0x3FFFu) << 16;
    d |= static_cast<uint64_t>((group >> 4) & 0x3FFFu) << 32;
    d |= static_cast<uint64_t>(1u) << 46;
    d |= static_cast<uint64_t>(2u) << 61;
    return d;
}
constexpr uint32_t kBTransposed = 1u << 16;  // instruction descriptor: B is MN-major

// lo += x's low bf16, hi += its high one
__device__ __forceinline__ void add_bf2(float& lo, float& hi, uint32_t x) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tadd.rn.f32.bf16 %0, a, %0;\n\tadd.rn.f32.bf16 %1, b, %1;\n\t}"
        : "+f"(lo), "+f"(hi)
        : "r"(x));
}
__device__ __forceinline__ uint32_t pack_bf2(float lo, float hi) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&b);
}

__device__ __forceinline__ uint32_t elect_one() {
    uint32_t on;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(on));
    return on;
}
// One arrival of this thread on `bar` once all its copies so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
// A bounded wait of a whole warp, with one answer for all its lanes.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, int* err) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, kTimeout));
}
// Barrier `id` of `threads` threads, with the conjunction of what they bring.
__device__ __forceinline__ bool meet_all(int id, int threads, bool ok) {
    int all;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.s32 p, %1, 0;\n\tbar.red.and.pred q, %2, %3, p;\n\tselp.s32 %0, 1, 0, q;\n\t}"
        : "=r"(all)
        : "r"(ok ? 1 : 0), "r"(id), "r"(threads)
        : "memory");
    return all != 0;
}
__device__ __forceinline__ bool value_warps(bool ok) { return meet_all(1, kValueThreads, ok); }
// Bit i: the row at position pos sees key j0 + i, below `end`.
__device__ __forceinline__ uint32_t low_bits(int n) {  // the n lowest bits, n of any sign and size
    return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u;
}
__device__ __forceinline__ uint32_t seen_bits(int j0, int end, int pos, int window, int sinks) {
    uint32_t bits = low_bits(pos + 1 - j0);
    if (window > 0) bits &= ~low_bits(max(pos - window + 1, 0) - j0) | low_bits(sinks - j0);
    return bits & low_bits(end - j0);
}

// Tensor copies: the page of box `b` of `boxes` of a key tile, -1 for none (behind the range, or a bad page).
__device__ __forceinline__ int box_page(const PagedAttention& p, int s, const KeyTiles& kt, int tile, int b, int boxes, int box) {
    int start, end;
    key_range(kt, tile, kKeys, start, end);
    const int key = start + b * box;
    if (b >= boxes || key >= end) return -1;
    const int slot = page_slot(p, key);
    const int page = slot < p.batch.table_width ? p.batch.table[s * p.batch.table_stride + slot] : -1;
    return page < p.cache.pages ? page : -1;
}
// cp.async: offsets of the keys t, t + THREADS, .. of a key tile, and the copy of `keys` keys and `count` slabs from
// `slab` into [block of keys][slab][key] at dst.
template <int THREADS>
__device__ __forceinline__ void tile_offsets(const PagedAttention& p, int s, const KeyTiles& kt, int tile, int t,
                                             long long (&o)[kKeys / THREADS]) {
    int start, end;
    key_range(kt, tile, kKeys, start, end);
#pragma unroll
    for (int x = 0; x < kKeys / THREADS; ++x) {
        const int key = start + t + x * THREADS;
        o[x] = key < end ? key_offset(p, s, key) : -1;
    }
}
template <int THREADS>
__device__ __forceinline__ void copy_rows(uint32_t dst, const bf16* src, const long long* of, int keys, int block, int block_slabs,
                                          int slab, int count, int D, int t) {
    for (int x = 0; x < count; ++x) {
        const int d = (slab + x) * 64 + (t & 7) * 8;
#pragma unroll 4
        for (int key = t >> 3; key < keys; key += THREADS / 8) {
            const long long off = of[key];
            const bool in = off >= 0 && d < D;
            const int row = key & (block - 1);
            cp_async16(dst + (key - row) * (block_slabs * 128) + x * (block * 128) + row * 128 + (((t & 7) ^ (row & 7)) << 4),
                       in ? src + off + d : src, in);
        }
    }
}

// Values that are not finite, in a tile that not every row sees whole, would reach the rows that do not see them as 0 * v:
// zeros take their place in `count` keys from `first` of tile j, before the products read them, and the rows that see them
// get them at the end (*found is set). Keys from `end` on, and those of bad pages, are zeros outright (a tensor copy brought
// what lies there). Keys that every row of kt sees are left alone. By THREADS threads: with two threads per row by those,
// each the keys of its own scores, before they hand P over; with one by the value warps, since the registers are missing
// in the softmax (2048 tokens after 8192, head size 128: 202 us there, 175 here; head size 256: 310 there, 339 here).
template <int DP, int THREADS>
__device__ __forceinline__ void clean_values(const PagedAttention& p, int s, const KeyTiles& kt, unsigned char* ring, int* found,
                                             int j, int start, int end, int first, int count, int block, bool bad_page) {
    using Sh = TcShape<DP>;
    constexpr int kSlabs = Sh::kSlabs;
    const int t = threadIdx.x % THREADS, slabs = (p.cache.D + 63) / 64;
#pragma unroll 1
    for (int key = first + (t >> 3); key < first + count; key += THREADS / 8) {
        const int at = start + key, in = key % Sh::kPieceKeys, row = in & (block - 1);
        const bool absent = at >= end || (bad_page && key_offset(p, s, at) < 0);
        if (!absent && at <= kt.pmin && (p.window <= 0 || at < p.sinks || at > kt.pmax - p.window)) continue;
        uint4* w = reinterpret_cast<uint4*>(ring + ((j * Sh::kPieces + key / Sh::kPieceKeys) % Sh::kVRing) * Sh::kPieceBytes +
                                            (in - row) * (kSlabs * 128) + row * 128 + (((t & 7) ^ (row & 7)) << 4));
        const int step = block * (128 / 16);  // from slab to slab
        uint4 c[kSlabs];
#pragma unroll
        for (int x = 0; x < kSlabs; ++x) c[x] = x < slabs && !absent ? w[x * step] : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int x = 0; x < kSlabs; ++x) {
            uint32_t e[4] = {c[x].x, c[x].y, c[x].z, c[x].w}, top = 0;
            // an exponent of all ones carries into the bit above it
#pragma unroll
            for (int y = 0; y < 4; ++y) top |= (e[y] & 0x7f807f80u) + 0x00800080u;
            const bool bad = (top & 0x80008000u) != 0;
            if (bad) {
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    if ((e[y] & 0x7f80u) == 0x7f80u) e[y] &= 0xffff0000u;
                    if ((e[y] & 0x7f800000u) == 0x7f800000u) e[y] &= 0x0000ffffu;
                }
                *found = 1;
            }
            if (x < slabs && (bad || absent)) w[x * step] = make_uint4(e[0], e[1], e[2], e[3]);
        }
    }
}

template <int DP, bool CAP>
__global__ void __launch_bounds__(kThreads, 1) paged_tc_kernel(const __grid_constant__ Args a,
                                                               const __grid_constant__ CUtensorMap k_map,
                                                               const __grid_constant__ CUtensorMap v_map, const int k_box,
                                                               const int v_box) {
    using Sh = TcShape<DP>;
    constexpr int BN = kKeys, NK = Sh::kKRing, NV = Sh::kVRing, kPieces = Sh::kPieces, kSlabs = Sh::kSlabs;
    constexpr int kParts = Sh::kParts, kCols = Sh::kCols;
    constexpr bool kSumRounded = DP > 64;
    constexpr int kEarly = kParts == 1 ? 3 : 2;  // quarters of a tile's P handed over before the rest
    extern __shared__ unsigned char smem_raw[];
    const PagedAttention& p = a.p;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, D = p.cache.D;
    const int tile = a.row_tiles - 1 - static_cast<int>(blockIdx.x % a.row_tiles);
    const int rest = blockIdx.x / a.row_tiles, split = rest % a.splits, s = rest / a.splits, kvh = blockIdx.y;
    cudaTriggerProgrammaticLaunchCompletion();  // the join's blocks may take their places
    const Sequence sq = sequence(p, s, blockIdx.x % (a.row_tiles * a.splits) == 0 && kvh == 0 && tid == 0);
    const int rr0 = tile * Sh::kRows, n_rows = sq.n_new * a.G;
    if (!sq.ok || rr0 >= n_rows) return;
    const KeyTiles kt = key_tiles(sq.past, sq.n_new, a.G, rr0, rr0 + Sh::kRows, p.window, p.sinks, BN, a.align);
    const int t0 = split * a.split_tiles, n = min(kt.n, t0 + a.split_tiles) - t0;
    if (n <= 0) return;
    const bool partial = kt.n > a.split_tiles;
    const bool pair = Sh::kTiles == 2 && rr0 + 128 < n_rows;
    const bool tma = k_box > 0;

    // shared memory, 1024-byte aligned for the swizzle
    const uint32_t q_s = (smem_u32(smem_raw) + 1023u) & ~1023u;
    unsigned char* sm = smem_raw + (q_s - smem_u32(smem_raw));
    const uint32_t k_ring = q_s + Sh::kQBytes, v_ring = q_s + Sh::kVRingAt;
    const uint32_t bars = q_s + Sh::kBars;
    auto k_full = [&](int i) { return bars + 8u * i; };
    auto k_empty = [&](int i) { return bars + 8u * (NK + i); };
    auto v_full = [&](int i) { return bars + 8u * (2 * NK + i); };
    auto v_empty = [&](int i) { return bars + 8u * (2 * NK + NV + i); };
    auto s_full = [&](int i) { return bars + 8u * (2 * NK + 2 * NV + i); };
    auto p_early = [&](int i) { return bars + 8u * (2 * NK + 2 * NV + 2 + i); };
    auto p_full = [&](int i) { return bars + 8u * (2 * NK + 2 * NV + 4 + i); };
    auto pv_done = [&](int i) { return bars + 8u * (2 * NK + 2 * NV + 6 + i); };
    const uint32_t drained = bars + 8u * (2 * NK + 2 * NV + 8), q_full = drained + 8u, v_raw = q_full + 8u;
    int* words = reinterpret_cast<int*>(sm + Sh::kBars + Sh::kBarriers * 8);  // [0] tensor memory, [1] not finite

    if (warp == kMmaWarp) {
        tmem_alloc(smem_u32(words), 512);
        tmem_relinquish();
    }
    if (tid == 0) {
        for (int i = 0; i < NK; ++i) {
            mbar_init(k_full(i), tma ? 1 : 32);
            mbar_init(k_empty(i), 1);
        }
        for (int i = 0; i < NV; ++i) {
            mbar_init(v_full(i), tma ? 1 : kValueThreads);
            mbar_init(v_empty(i), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(s_full(i), 1);
            mbar_init(p_early(i), 4);
            mbar_init(p_full(i), 4);
            mbar_init(pv_done(i), 1);
        }
        mbar_init(drained, 1);
        mbar_init(v_raw, 1);
        mbar_init(q_full, kSoftmaxWarps * 32);
        fence_barrier_init();
        words[1] = 0;
    }
    const bool bad_here = any_bad_page(p, s, kt, t0, n, BN);
    tc_fence_before();
    const bool bad_page = __syncthreads_or(bad_here);  // (and the barriers and words[] are set)
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(words);
    float* maxima = reinterpret_cast<float*>(sm + Sh::kMax);
    // a softmax thread's row tile, part of the row, and row; tensor memory lanes 32 (warp & 3) ..
    const int rt = kParts == 1 ? warp >> 2 : 0, part = kParts == 1 ? 0 : warp >> 2, my_rr = rr0 + rt * 128 + (tid & 127);
    const int my_pos = my_rr < n_rows ? sq.past + head_group(a, my_rr) : -1;
    const uint32_t my_lanes = tmem + (static_cast<uint32_t>(warp & 3) << 21);
    const bool softmax_on = warp < kSoftmaxWarps && (kParts > 1 || rt == 0 || pair);
    float m = -INFINITY, l = 0.f;
    const int v_block = kPieces > 1 && tma ? v_box : Sh::kBlock;  // keys of a block of V

    if (warp < kSoftmaxWarps) {
        // Q, by the softmax warps, which have nothing else to do yet; only the issuing warp waits for it
        {
            constexpr int kChunks = DP / 8, kRowsPerPass = kSoftmaxWarps * 32 / kChunks;
            const bf16* q = static_cast<const bf16*>(p.q);
            const int rows = pair ? 256 : 128, c = tid % kChunks;
#pragma unroll 4
            for (int r = tid / kChunks; r < rows; r += kRowsPerPass) {
                const int rr = rr0 + r, t = head_group(a, rr), lr = r & 127;
                const bool in = rr < n_rows && c * 8 < D;
                const bf16* src = in ? q + (sq.row0 + t) * p.ldq + static_cast<long long>(kvh * a.G + rr - t * a.G) * D + c * 8 : q;
                cp_async16(q_s + (r >> 7) * (128 * DP * 2) + (c >> 3) * (128 * 128) + lr * 128 + (((c & 7) ^ (lr & 7)) << 4), src, in);
            }
        }
        cp_async_commit();
        cp_async_wait<0>();
        fence_proxy_async_smem();
        mbar_arrive(q_full);
        if (softmax_on) {
            const float scale_log2 = p.scale * kLog2e;
            const float cap_in = CAP ? 2.f * scale_log2 / p.softcap : 0.f, cap_out = p.softcap * kLog2e;
            // positions of this row tile
            KeyTiles mine = kt;
            mine.pmin = sq.past + (rr0 + rt * 128) / a.G;
            mine.pmax = sq.past + (min(n_rows, rr0 + rt * 128 + 128) - 1) / a.G;
            const uint32_t o_t = my_lanes + Sh::kO + rt * DP;
            bool ok = true;
            for (int j = 0; j < n; ++j) {
                const int slot = pair ? rt : j & 1, turn = pair ? j : j >> 1;
                int start, end;
                key_range(kt, t0 + j, BN, start, end);
                const bool whole = end - start == BN && !bad_page && all_seen(mine, start, end, p.window, p.sinks);
                const uint32_t s_t = my_lanes + slot * BN;
                ok = ok && warp_wait(s_full(slot), turn & 1, p.err);
                if (kParts == 1 && !ok) break;
                // this thread's scores in registers: the loads are in flight together
                uint32_t x[kCols];
                float mx = -INFINITY;
                if (ok) {
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < kCols / 32; ++c) tmem_ld32(s_t + part * kCols + c * 32, &x[c * 32]);
                    tmem_wait_ld();
                    if (!whole) {
#pragma unroll
                        for (int c = 0; c < kCols / 32; ++c) {
                            const int j0 = start + part * kCols + c * 32;
                            uint32_t bits = seen_bits(j0, end, my_pos, p.window, p.sinks);
                            if (bad_page) {
                                for (int i = 0; i < 32; ++i)
                                    if ((bits >> i & 1u) && key_offset(p, s, j0 + i) < 0) bits &= ~(1u << i);
                            }
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (!(bits & (1u << i))) x[c * 32 + i] = 0xff800000u;
                        }
                    }
                    float mx4[4];
#pragma unroll
                    for (int c = 0; c < 4; ++c) mx4[c] = fmaxf(__uint_as_float(x[c]), __uint_as_float(x[4 + c]));
#pragma unroll
                    for (int i = 8; i < kCols; i += 4)
#pragma unroll
                        for (int c = 0; c < 4; ++c) mx4[c] = fmaxf(mx4[c], __uint_as_float(x[i + c]));
                    mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
                }
                if constexpr (kParts > 1) {
                    // The row's threads agree on its maximum; they have read their scores by then, so that P may be
                    // written over them. After a failed wait they leave together.
                    float* const my_max = maxima + (j & 1) * (kParts * 128) + (tid & 127);
                    my_max[part * 128] = mx;
                    ok = meet_all(2 + (warp & 3), kParts * 32, ok);
                    if (!ok) break;
                    mx = fmaxf(my_max[0], my_max[128]);
                }
                // both maps rise with the score (scale > 0), so the maximum is mapped alone
                if (mx != -INFINITY) mx = CAP ? soft_cap_log2(mx, cap_in, cap_out) : mx * scale_log2;
                const bool move = mx > m + 8.f;  // (-inf + 8 is passed by any score)
                if (__any_sync(0xffffffffu, move)) {
                    const float alpha = move ? ex2_approx(m - mx) : 1.f;
                    m = move ? mx : m;
                    l *= alpha;
                    if (j > 0) {  // O holds sums against the old reference; each part rescales some of its channels
                        const int slot0 = pair ? rt : (j - 1) & 1, turn0 = pair ? j - 1 : (j - 1) >> 1;
                        ok = warp_wait(pv_done(slot0), turn0 & 1, p.err);
                        if (ok) {
                            tc_fence_after();
                            for (int c = part * 16; c < D; c += kParts * 16) {
                                uint32_t r[16];
                                tmem_ld16(o_t + c, r);
                                tmem_wait_ld();
#pragma unroll
                                for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
                                tmem_st16(o_t + c, r);
                            }
                        }
                        if constexpr (kParts > 1) {
                            // The products that start on p_early, which part 0 alone hands over, add to every channel: they
                            // start after both parts' rescaling. The parts hold the same m and maximum, so that both or
                            // neither come here. (An arrival of part 1 on p_early in every tile cost 1 to 2 % more.)
                            tmem_wait_st();
                            tc_fence_before();
                            ok = meet_all(2 + (warp & 3), kParts * 32, ok);
                            tc_fence_after();
                        }
                        if (!ok) continue;  // (to tell the row's other threads, or to leave)
                    }
                }
                const float ref = m == -INFINITY ? 0.f : m;
                const uint64_t k2 = f2_make(scale_log2, scale_log2), r2 = f2_make(-ref, -ref);
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
                uint64_t sum2[2] = {0, 0};
#pragma unroll
                for (int c = 0; c < kCols / 32; ++c) {
                    uint32_t pk[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float x0 = __uint_as_float(x[c * 32 + 2 * i]), x1 = __uint_as_float(x[c * 32 + 2 * i + 1]);
                        uint64_t e;
                        if constexpr (CAP) {
                            e = add2(f2_make(soft_cap_log2(x0, cap_in, cap_out), soft_cap_log2(x1, cap_in, cap_out)), r2);
                            const float2 v = f2_split(e);  // the cap maps what is masked to a number: it stays masked
                            if (!whole) e = f2_make(x0 == -INFINITY ? x0 : v.x, x1 == -INFINITY ? x1 : v.y);
                        } else {
                            e = fma2(f2_make(x0, x1), k2, r2);
                        }
                        const float2 v = f2_split(e);
                        const float e0 = ex2_approx(v.x), e1 = ex2_approx(v.y);
                        pk[i] = pack_bf2(e0, e1);
                        if (kSumRounded) add_bf2(sum[(2 * i) & 3], sum[(2 * i + 1) & 3], pk[i]);
                        else sum2[i & 1] = add2(sum2[i & 1], f2_make(e0, e1));
                    }
                    tmem_st16(s_t + part * (kCols / 2) + c * 16, pk);  // over the scores, which this row has read
                    if (kParts == 1 && c == kEarly - 1) {              // the products over these keys may start
                        tmem_wait_st();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(p_early(slot));
                    }
                }
                const float2 total = f2_split(add2(sum2[0], sum2[1]));
                l += kSumRounded ? (sum[0] + sum[1]) + (sum[2] + sum[3]) : total.x + total.y;
                if (kParts > 1 && !whole) {  // the values of this part's keys
                    for (int pc = part * (kPieces / kParts); pc < (part + 1) * kPieces / kParts && ok; ++pc) {
                        const int g = j * kPieces + pc;
                        ok = warp_wait(v_full(g % NV), (g / NV) & 1, p.err);
                    }
                    if (!ok) continue;  // (as above)
                    clean_values<DP, 128>(p, s, mine, sm + Sh::kVRingAt, words + 1, j, start, end, part * kCols, kCols,
                                          v_block, bad_page);
                    fence_proxy_async_smem();
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(kParts == 1 || part == 1 ? p_full(slot) : p_early(slot));
            }
        }
    } else if (warp == kKeyWarp) {
        const int slabs = (D + 63) / 64;
        auto piece_slabs = [&](int pc) { return min(Sh::kPieceSlabs, max(0, slabs - pc * Sh::kPieceSlabs)); };
        bool ok = true;
        if (tma) {
            // lane b < BN / k_box holds the page of box b, `k_box` keys of one page; one elected thread copies
            const int boxes = BN / k_box;
            auto page_of = [&](int j) { return box_page(p, s, kt, t0 + j, lane, boxes, k_box); };
            const bool leader = elect_one() != 0;
            int next = page_of(0), issued = 0;
            for (int j = 0; j < n && ok; ++j) {
                const int page = next;
                if (j + 1 < n) next = page_of(j + 1);
                int start, end;
                key_range(kt, t0 + j, BN, start, end);
                const int at = start + lane * k_box - page_slot(p, start + lane * k_box) * p.cache.page_size;
                const uint32_t box_bytes = static_cast<uint32_t>(__popc(__ballot_sync(0xffffffffu, page >= 0))) * k_box * 128;
                for (int pc = 0; pc < kPieces && ok; ++pc) {
                    const int g = j * kPieces + pc, slot = g % NK, count = piece_slabs(pc);
                    ok = warp_wait(k_empty(slot), ((g / NK) & 1) ^ 1, p.err);
                    if (!ok) continue;
                    if (leader) mbar_arrive_expect_tx(k_full(slot), box_bytes * count);
                    __syncwarp();
                    const uint32_t dst = k_ring + slot * Sh::kPieceBytes;
                    for (int b = 0; b < boxes; ++b) {
                        const int pg = __shfl_sync(0xffffffffu, page, b), row = __shfl_sync(0xffffffffu, at, b);
                        if (leader && pg >= 0)
                            for (int x = 0; x < count; ++x)
                                tma_load_4d(&k_map, dst + x * (BN * 128) + b * k_box * 128, k_full(slot),
                                            (pc * Sh::kPieceSlabs + x) * 64, row, kvh, pg);
                    }
                    issued = g + 1;
                }
            }
            if (!ok)  // what is on its way lands (or is waited for as long as a wait may last) before the block ends
                for (int g = issued > NK ? issued - NK : 0; g < issued; ++g) mbar_wait_quiet(k_full(g % NK), (g / NK) & 1);
        } else {
            const bf16* kc = static_cast<const bf16*>(p.cache.k) + kvh * p.cache.head_stride;
            long long* offs = reinterpret_cast<long long*>(sm + Sh::kOffs);
            long long next[4];
            tile_offsets<32>(p, s, kt, t0, lane, next);
            for (int j = 0; j < n && ok; ++j) {
                long long* of = offs + (j & 1) * BN;
#pragma unroll
                for (int x = 0; x < 4; ++x) of[lane + x * 32] = next[x];
                __syncwarp();
                if (j + 1 < n) tile_offsets<32>(p, s, kt, t0 + j + 1, lane, next);
                for (int pc = 0; pc < kPieces && ok; ++pc) {
                    const int g = j * kPieces + pc, slot = g % NK;
                    ok = warp_wait(k_empty(slot), ((g / NK) & 1) ^ 1, p.err);
                    if (!ok) continue;
                    copy_rows<32>(k_ring + slot * Sh::kPieceBytes, kc, of, BN, BN, Sh::kPieceSlabs, pc * Sh::kPieceSlabs,
                                  piece_slabs(pc), D, lane);
                    cp_async_arrive(k_full(slot));
                }
            }
            cp_async_commit();
            cp_async_wait<0>();
        }
    } else if (warp < kMmaWarp) {
        constexpr bool kClean = kParts == 1;
        const int pt = tid - kValueWarp * 32, slabs = (D + 63) / 64;
        auto is_edge = [&](int start, int end) {
            return kClean && (end - start < BN || bad_page || !all_seen(kt, start, end, p.window, p.sinks));
        };
        bool ok = true;
        if (tma) {
            // as for K, by the first value warp; the second helps to clean and keeps step, waiting for no place
            const int boxes = BN / v_box, boxes_piece = Sh::kPieceKeys / v_box;
            auto page_of = [&](int j) { return box_page(p, s, kt, t0 + j, lane, boxes, v_box); };
            const bool leader = elect_one() != 0, all_slabs = kPieces > 1 && D % 64 == 0;
            int next = page_of(0), issued = 0, raw = 0;
            bool in_flight = false;  // on v_raw
            for (int j = 0; j < n; ++j) {
                const int page = next;
                if (j + 1 < n) next = page_of(j + 1);
                int start, end;
                key_range(kt, t0 + j, BN, start, end);
                const int at = start + lane * v_box - page_slot(p, start + lane * v_box) * p.cache.page_size;
                const unsigned there = __ballot_sync(0xffffffffu, page >= 0);
                const uint32_t box_bytes = static_cast<uint32_t>(v_box) * 128 * slabs;
                const bool edge = is_edge(start, end);
                for (int pc = 0; pc < kPieces && ok && warp == kValueWarp; ++pc) {
                    const int g = j * kPieces + pc, slot = g % NV;
                    ok = warp_wait(v_empty(slot), ((g / NV) & 1) ^ 1, p.err);
                    if (!ok) continue;
                    const uint32_t bar = edge ? v_raw : v_full(slot);
                    const unsigned mine = there >> (pc * boxes_piece) & ((1u << boxes_piece) - 1u);
                    if (leader) mbar_arrive_expect_tx(bar, __popc(mine) * box_bytes);
                    __syncwarp();
                    uint32_t dst = v_ring + slot * Sh::kPieceBytes;
                    for (int b = pc * boxes_piece; b < (pc + 1) * boxes_piece; ++b, dst += v_box * (kPieces > 1 ? kSlabs * 128 : 128)) {
                        const int pg = __shfl_sync(0xffffffffu, page, b), row = __shfl_sync(0xffffffffu, at, b);
                        if (leader && pg >= 0) {
                            if (all_slabs) {
                                tma_load_5d(&v_map, dst, bar, 0, row, 0, kvh, pg);
                            } else {
                                for (int x = 0; x < slabs; ++x) tma_load_4d(&v_map, dst + x * (v_block * 128), bar, x * 64, row, kvh, pg);
                            }
                        }
                    }
                    if (edge) in_flight = true;
                    else issued = g + 1;
                }
                if (!kClean) {
                    if (!ok || warp != kValueWarp) break;
                    continue;
                }
                ok = value_warps(ok);
                if (!ok) break;
                if (!edge) continue;
                ok = value_warps(warp_wait(v_raw, raw & 1, p.err));
                if (!ok) break;
                in_flight = false;
                ++raw;
                clean_values<DP, kValueThreads>(p, s, kt, sm + Sh::kVRingAt, words + 1, j, start, end, 0, BN, v_block, bad_page);
                fence_proxy_async_smem();
                value_warps(true);
                if (pt == 0) mbar_arrive(v_full(j % NV));
                issued = j + 1;
            }
            if (!ok && warp == kValueWarp) {
                if (in_flight) mbar_wait_quiet(v_raw, raw & 1);
                for (int g = issued > NV ? issued - NV : 0; g < issued; ++g) mbar_wait_quiet(v_full(g % NV), (g / NV) & 1);
            }
        } else {
            const bf16* vc = static_cast<const bf16*>(p.cache.v) + kvh * p.cache.head_stride;
            long long* offs = reinterpret_cast<long long*>(sm + Sh::kOffs) + 2 * BN;
            long long next[2];
            tile_offsets<kValueThreads>(p, s, kt, t0, pt, next);
            for (int j = 0; j < n; ++j) {
                long long* of = offs + (j & 1) * BN;
#pragma unroll
                for (int x = 0; x < 2; ++x) of[pt + x * kValueThreads] = next[x];
                ok = value_warps(ok);  // after a failed wait the warps leave together
                if (!ok) break;
                if (j + 1 < n) tile_offsets<kValueThreads>(p, s, kt, t0 + j + 1, pt, next);
                int start, end;
                key_range(kt, t0 + j, BN, start, end);
                const bool edge = is_edge(start, end);
                for (int pc = 0; pc < kPieces && ok; ++pc) {
                    const int g = j * kPieces + pc, slot = g % NV;
                    ok = warp_wait(v_empty(slot), ((g / NV) & 1) ^ 1, p.err);
                    if (!ok) continue;
                    copy_rows<kValueThreads>(v_ring + slot * Sh::kPieceBytes, vc, of + pc * Sh::kPieceKeys, Sh::kPieceKeys, Sh::kBlock, kSlabs, 0,
                                             slabs, D, pt);
                    if (!edge) cp_async_arrive(v_full(slot));
                }
                if (!edge || !ok) continue;
                cp_async_commit();
                cp_async_wait<0>();
                ok = value_warps(true);  // both warps' copies are there (what a thread cleans, another may have copied)
                clean_values<DP, kValueThreads>(p, s, kt, sm + Sh::kVRingAt, words + 1, j, start, end, 0, BN, v_block, bad_page);
                mbar_arrive(v_full(j % NV));
            }
            cp_async_commit();
            cp_async_wait<0>();
        }
    } else {
        // The whole warp walks the tiles, so that all it computes is uniform; one elected thread issues.
        const int d16 = (D + 15) & ~15, k_steps = d16 / 16;
        const uint32_t t_mem = __shfl_sync(0xffffffffu, tmem, 0);
        const uint32_t idesc_s = idesc_bf16_f32(128, BN);
        const uint32_t idesc_o = idesc_bf16_f32(128, d16) | kBTransposed;
        // descriptors of the first operands; the others differ in the address field alone (16-byte units)
        const uint64_t q_desc = kmajor_sw128_desc(q_s), k_desc = kmajor_sw128_desc(k_ring);
        const uint64_t v_desc = mnmajor_sw128_desc(v_ring, v_block * 128, v_block == 8 ? kSlabs * 1024 : 1024);
        const uint32_t leader = elect_one();
        auto piece_there = [&](uint32_t bar, int turn) -> bool {
            if (!warp_wait(bar, turn & 1, p.err)) return false;
            // cp.async writes through the generic proxy, the products read through the async one: ordered here, by
            // the threads that have seen the copies land
            if (!tma) fence_proxy_async_smem();
            tc_fence_after();
            return true;
        };
        // The products of a tile in one piece are branched around by the other lanes, those of smaller pieces predicated:
        // 170 and 183 us, but 370 and 350 us (2048 tokens after 8192, head sizes 128 and 256).
        constexpr bool kBranch = kPieces == 1;
        const uint32_t on = kBranch ? 1u : leader;
        // unit u: key tile j of row tile t, in slot u & 1; the second row tile reads what the first has waited for
        auto walk = [&](auto two) {
            constexpr bool kPair = decltype(two)::value;
            auto scores = [&](int u, int slot) -> bool {
                const int j = kPair ? u >> 1 : u, t = kPair ? slot : 0;
                for (int pc = 0; pc < kPieces; ++pc) {
                    const int g = j * kPieces + pc, at = g % NK;
                    if ((!kPair || t == 0) && !piece_there(k_full(at), g / NK)) return false;
                    const uint64_t kd = k_desc + static_cast<uint64_t>(at * Sh::kPieceBytes >> 4);
                    const uint64_t qd = q_desc + static_cast<uint64_t>((t * (128 * DP * 2) + pc * Sh::kPieceSlabs * (128 * 128)) >> 4);
                    auto step = [&](int k) {
                        umma_ss(t_mem + slot * BN, qd + (((k >> 2) * (128 * 128) + (k & 3) * 32) >> 4),
                                kd + (((k >> 2) * (BN * 128) + (k & 3) * 32) >> 4), idesc_s, k > 0 || pc > 0, on);
                    };
                    const int steps = min(4 * Sh::kPieceSlabs, k_steps - pc * 4 * Sh::kPieceSlabs);
                    if (!kBranch || leader) {
                        if (steps == 4 * Sh::kPieceSlabs) {
#pragma unroll
                            for (int k = 0; k < 4 * Sh::kPieceSlabs; ++k) step(k);
                        } else {
                            for (int k = 0; k < steps; ++k) step(k);
                        }
                    }
                    __syncwarp();
                    if (pc == kPieces - 1) umma_commit_on(s_full(slot), leader);
                    if (!kPair || t == 1) umma_commit_on(k_empty(at), leader);
                }
                return true;
            };
            auto values = [&](int u, int slot) -> bool {
                const int j = kPair ? u >> 1 : u, t = kPair ? slot : 0;
                const uint32_t o = t_mem + Sh::kO + t * DP, pa = t_mem + slot * BN;
                constexpr int kSteps = BN / 16 / kPieces;
                for (int pc = 0; pc < kPieces; ++pc) {
                    const int g = j * kPieces + pc, at = g % NV;
                    if ((!kPair || t == 0) && !piece_there(v_full(at), g / NV)) return false;
                    const uint64_t vd = v_desc + static_cast<uint64_t>(at * Sh::kPieceBytes >> 4);
                    auto step = [&](int k) {  // 16 keys
                        umma_ts(o, pa + (pc * kSteps + k) * 8, vd + (k * (kPieces > 1 ? 2048 * kSlabs : 2048) >> 4), idesc_o,
                                k > 0 || pc > 0 || j > 0, on);
                    };
                    // quarters of P that are handed over early, and the rest
                    constexpr int kQuarters = 4 / kPieces;  // of a piece
                    if (pc == 0) {
                        if (!warp_wait(p_early(slot), (u >> 1) & 1, p.err)) return false;
                        tc_fence_after();
                    }
                    if (kPieces == 1) {
                        if (!kBranch || leader) {
#pragma unroll
                            for (int k = 0; k < 2 * kEarly; ++k) step(k);
                        }
                        __syncwarp();
                    }
                    if (pc * kQuarters == kEarly || kPieces == 1) {
                        if (!warp_wait(p_full(slot), (u >> 1) & 1, p.err)) return false;
                        tc_fence_after();
                    }
                    if (!kBranch || leader) {
#pragma unroll
                        for (int k = kPieces == 1 ? 2 * kEarly : 0; k < kSteps; ++k) step(k);
                    }
                    __syncwarp();
                    if (pc == kPieces - 1) umma_commit_on(pv_done(slot), leader);
                    if (!kPair || t == 1) umma_commit_on(v_empty(at), leader);
                }
                return true;
            };
            const int units = kPair ? 2 * n : n;
            bool ok = warp_wait(q_full, 0, p.err) && scores(0, 0) && (units < 2 || scores(1, 1));
            for (int u = 0; u < units && ok; u += 2) {
                ok = values(u, 0) && (u + 2 >= units || scores(u + 2, 0));
                if (ok && u + 1 < units) ok = values(u + 1, 1) && (u + 3 >= units || scores(u + 3, 1));
            }
        };
        if (Sh::kTiles == 2 && pair) walk(std::true_type{});
        else walk(std::false_type{});
        umma_commit_on(drained, leader);  // whatever was issued has run before the tensor memory is given back
        mbar_wait_quiet(drained, 0);
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();

    if (kParts > 1) {  // the sums of a row's threads meet where the maxima were
        if (softmax_on) maxima[part * 128 + (tid & 127)] = l;
        __syncthreads();
        if (softmax_on) l = maxima[tid & 127] + maxima[128 + (tid & 127)];
    }
    if (softmax_on) {
        const long long row = sq.row0 + my_rr / a.G;
        const int h = kvh * a.G + my_rr % a.G;
        const bool live = my_rr < n_rows;
        const long long at = (static_cast<long long>(split) * p.batch.rows + row) * p.q_heads + h;
        const float inv = partial ? 1.f : (l == 0.f ? 0.f : 1.f / l);
        if (partial && live && part == 0) a.ml[at] = make_float2(m, l);
        const bool repair = *reinterpret_cast<volatile int*>(words + 1) != 0;
        bf16* out = static_cast<bf16*>(p.out) + row * p.ldo + static_cast<long long>(h) * D;
        for (int c = part * 32; c < D; c += kParts * 32) {
            uint32_t r[32];
            tmem_ld32(my_lanes + Sh::kO + rt * DP + c, r);
            tmem_wait_ld();
            float o[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __uint_as_float(r[i]) * inv;
            if (repair && live) {
                const bf16* vc = static_cast<const bf16*>(p.cache.v) + kvh * p.cache.head_stride;
                for (int t = 0; t < n; ++t) {
                    int start, end;
                    key_range(kt, t0 + t, BN, start, end);
                    if (all_seen(kt, start, end, p.window, p.sinks)) continue;
                    for (int j = start; j < end; ++j) {
                        if (!seen(j, my_pos, p.window, p.sinks)) continue;
                        const long long off = key_offset(p, s, j);
                        if (off < 0) continue;
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            if (c + i >= D) continue;
                            const float v = __bfloat162float(vc[off + c + i]);
                            if ((__float_as_uint(v) & 0x7f800000u) == 0x7f800000u) o[i] += v;
                        }
                    }
                }
            }
            if (!live) continue;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                if (c + 8 * b >= D) continue;
                const float* x = o + 8 * b;
                if (partial) {
                    float4* dst = reinterpret_cast<float4*>(a.part + at * D + c + 8 * b);
                    dst[0] = make_float4(x[0], x[1], x[2], x[3]);
                    dst[1] = make_float4(x[4], x[5], x[6], x[7]);
                } else {
                    *reinterpret_cast<uint4*>(out + c + 8 * b) =
                        make_uint4(pack_bf2(x[0], x[1]), pack_bf2(x[2], x[3]), pack_bf2(x[4], x[5]), pack_bf2(x[6], x[7]));
                }
            }
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
}

template <int DP, bool CAP>
void launch(const Args& a, dim3 grid, cudaStream_t st) {
    static PerDeviceOnce once;
    using Sh = TcShape<DP>;
    static_assert(Sh::kSmem <= 232448, "shared memory of one block");
    if (once.pending()) {
        SANA_CUDA(cudaFuncSetAttribute(paged_tc_kernel<DP, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem));
        once.mark();
    }
    const int k_box = copy_box(a.p.cache, kKeys), v_box = k_box > 0 ? copy_box(a.p.cache, Sh::kBlock) : 0;
    CUtensorMap k{}, v{};
    if (k_box > 0) {
        k = pool_map(a.p.cache, a.p.cache.k, k_box);
        v = Sh::kPieces > 1 && a.p.cache.D % 64 == 0 ? pool_map_slabs(a.p.cache, a.p.cache.v, v_box) : pool_map(a.p.cache, a.p.cache.v, v_box);
    }
    paged_tc_kernel<DP, CAP><<<grid, kThreads, Sh::kSmem, st>>>(a, k, v, k_box, v_box);
}

}  // namespace

int tc_rows(int D) { return D <= 128 ? 256 : 128; }
int tc_keys() { return kKeys; }
void launch_tc(const Args& a, dim3 grid, cudaStream_t st) {
    const bool cap = a.p.softcap > 0.f;
    if (a.p.cache.D <= 64) cap ? launch<64, true>(a, grid, st) : launch<64, false>(a, grid, st);
    else if (a.p.cache.D <= 128) cap ? launch<128, true>(a, grid, st) : launch<128, false>(a, grid, st);
    else cap ? launch<256, true>(a, grid, st) : launch<256, false>(a, grid, st);
}

}  // namespace pattn
}  // namespace sana
