// attention.cu -- attention over packed sequences (openfish_b200_attention).
//
//   out[i] = sum_j p_ij v_j / sum_j p_ij,   p_ij = 2^(c <q_i, k_j> - m_i),   c = scale log2(e),
//
// in one pass over the keys: m_i is a running maximum, and what has been summed is scaled when it moves.
//
// A block takes the rows of one sequence and key head, 128 or two halves of 128, against the keys in tiles of 64.  The query
// heads that share a key head are rows next to each other (row r is query r / g, head r % g of the group), so that
// grouped heads and single tokens fill the same tiles and a key is read once for all of them.
//
//   4 warps to a half   the softmax, a thread to a row
//   1 warp to a half    the matrix instructions: S = Q K^T into tensor memory, O += P V with P read from there, in S's place
//   1 warp              asynchronous copies of the keys' and values' tiles (heads of up to 64: the last warp above)
//
// Tensor memory and registers decide how many halves there are to an SM, and only other halves' work fills the waits between a
// tile's steps.  Heads of up to 64: S and O take 128 columns, four blocks of a half, of 96 registers a thread (56 bytes
// do not fit and go through memory).  Heads of up to 128: O alone takes
// that, so two halves, each with two S in turn: the next tile's S is formed while this tile's weights are worked out.  The
// two share a block and its tiles, for the copies' way into shared memory and the products' way out of it are what bounds
// these heads: 48 cycles for each 128 x 64 x 16 of Q K^T (6 KB), 64 for 128 x 128 x 16 of P V.  Where there are rows for one half only (single
// tokens), a block has one, and an SM two blocks.
//
// Single tokens with one or two heads to a key head have no use for tiles of 128 rows: attention_few_kernel.
#include <math.h>
#include <stdint.h>

#include "encoder_device.cuh"
#include "tc5.cuh"

namespace {

using ofe::add2;
using ofe::fma2;
using ofe::pack;

__device__ int g_status;  // how many waits of the kernels have run out on this device
Reports g_reports;
thread_local int t_known[Reports::kDevices];

constexpr int kRows = 128;  // of a half
constexpr int kKeys = 64;   // of a tile
constexpr float kLazy = 8.f;  // a maximum may be outgrown by 2^8 before what has been summed is scaled
// Weights are held as 2^kRoom of their size.  The smallest number of fp16 is 2^-24 and its steps there are as large: without the room a key
// that the largest outweighs by more is lost or doubled (131072 keys of 2^-24.9 beside one of 1 whose value is zero: 0.0062 for 0.0033).  With
// it an underflow costs at most 2^-30 of a row's largest weight.  More room would leave less above, and a row whose first tile shows it few of its
// keys outgrows its maximum soon (windows of 257 keys, us with none, 5, 6, 7: 89.3, 89.7, 90.1, 91.4).
template <class T>
constexpr float kRoom = 5.f;
template <>
constexpr float kRoom<__nv_bfloat16> = 0.f;  // (goes down to 2^-133)
// What a tile's weights may add up to when they are worked out with the maximum there was before: none of them can be beyond the type.
constexpr float kMostOfTile = 65504.f;

struct Args {
    const int32_t *q_start, *k_start, *q_used, *k_used;
    const void *q, *k, *v;
    void *out;
    float *part, *part_lse;  // of a split: [split][sequences * max_q][q_heads][head_dim] and [split][sequences * max_q][q_heads]
    long long part_step;     // sequences * max_q * q_heads
    long long q_stride_row, q_stride_head, k_stride_row, k_stride_head, v_stride_row, v_stride_head, out_stride_row, out_stride_head;
    int q_rows, k_rows, q_heads, kv_heads, group, head_dim, sequences, max_q, max_k, left, right;
    ofe::Divider by_group;
    int tiles, splits;  // blocks of rows to the longest sequence; pieces of a block's keys
    float c;
    bool q_by_copy;    // the group divides a half's rows: a tiled copy brings the queries
    bool out_by_copy;  // it divides a warp's rows: and takes the results
};

// A sequence's rows in a tensor of `rows`, cut to the room there is.
__device__ __forceinline__ void span(const int32_t *start, const int32_t *used, int s, int rows, int most, int *first, int *count) {
    const int lo = min(max(start[s], 0), rows), hi = min(max(start[s + 1], lo), rows);
    int n = hi - lo;
    if (used) n = min(n, max(used[s], 0));
    *first = lo;
    *count = min(n, most);
}
// The keys that query i of nq sees of nk: [lo, hi).
__device__ __forceinline__ void window(const Args &a, int i, int nq, int nk, int *lo, int *hi) {
    const int place = i + nk - nq;
    *lo = a.left < 0 ? 0 : max(place - a.left, 0);
    *hi = a.right < 0 ? nk : min(place + a.right + 1, nk);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The largest of three numbers (a NaN is passed over).
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
// Two weights 2^(c s - c m + room) as the matrix unit takes them: its operands have 16 bits.  They are added to their row's sum in fp32, before they are
// rounded (a sum of the rounded ones would take two conversions more for every two keys, in the loop that bounds the kernel).
template <class T>
__device__ __forceinline__ uint32_t weights(float u, float w, float c, float shift, float2 &sum) {
    float2 z = {fmaf(u, c, shift), fmaf(w, c, shift)};
    z.x = ex2(z.x);
    z.y = ex2(z.y);
    sum = add2(sum, z);
    return pack<T>(z.x, z.y);
}

template <int DP, int H>
struct Shape {
    static constexpr int kBuffers = DP == 64 ? 1 : 2;           // S at a time
    static constexpr int kBlocks = (DP == 64 ? 4 : 2) / H;      // to an SM
    static constexpr int kChunks = DP / 64;                     // of 64 elements, 128 bytes
    static constexpr int kQueryBytes = kChunks * kRows * 128, kTileBytes = kChunks * kKeys * 128;
    // The ring moves in steps: step i brings the keys of tile i and the values of tile i - kBuffers, whose weights have the
    // place that tile i's S goes to.
    static constexpr int kStages = H == 2 ? 5 : 2, kStageBytes = 2 * kTileBytes;
    static constexpr bool kCopyWarp = DP == 128;                // a warp of its own for the copies, where registers allow one
    static constexpr int kThreads = 32 * (5 * H + kCopyWarp);
    static constexpr int kHalfBarriers = 2 * kBuffers + 3;      // s_full and p_ready of each S, q_ready, the last two o_done
    static constexpr int kBytes = H * kQueryBytes + kStages * kStageBytes + (2 * kStages + H * (kHalfBarriers + 2)) * 8 + 8;
    // columns of tensor memory, a power of two: S and O of each half
    static constexpr int kHalfColumns = kBuffers * kKeys + DP, kColumns = H * kHalfColumns, kOut = kBuffers * kKeys;
};

// Results beyond this are worked out again with weights in fp32.  A result is a mean of values, but by the tiles its weights are rounded to
// 16 bits one by one and their sum is not, so that among the type's largest numbers it may come out beyond them: an infinity.
template <class T>
constexpr float kLargest = 65504.f;
template <>
constexpr float kLargest<__nv_bfloat16> = 0x1.fep127f;

// One row again, by a warp, straight from its definition and reading only the keys that the row sees.  A matrix
// instruction multiplies the values of masked keys by weights of zero, which is no zero where such a value is an infinity or NaN.
template <class T>
__device__ __noinline__ float2 redo_row(const T *q, const T *k, const T *v, long long k_stride, long long v_stride, int head_dim, float c, int lo,
                                        int hi, float *out, T *out16) {
    const int lane = threadIdx.x & 31;
    float qf[4], acc[4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        qf[n] = lane + 32 * n < head_dim ? ofe::to_float(q[lane + 32 * n]) : 0.f;
        acc[n] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int j = lo; j < hi && l == l; ++j) {
        float z = 0.f;
#pragma unroll
        for (int n = 0; n < 4; ++n)
            if (lane + 32 * n < head_dim) z = fmaf(qf[n], ofe::to_float(k[j * k_stride + lane + 32 * n]), z);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) z += __shfl_xor_sync(0xffffffffu, z, d);
        const float next = fmaxf(m, z), from = next == -INFINITY ? 0.f : next;
        const float fade = m == next ? 1.f : ex2((m - next) * c), p = ex2((z - from) * c);
        m = next;
        l = l * fade + p;
#pragma unroll
        for (int n = 0; n < 4; ++n)
            if (lane + 32 * n < head_dim) acc[n] = fmaf(p, ofe::to_float(v[j * v_stride + lane + 32 * n]), acc[n] * fade);
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
        const int d = lane + 32 * n;
        if (d >= head_dim) continue;
        // a sum that is no number makes every element none (the loop ends there)
        const float f = l == l ? acc[n] / l : NAN;
        if (out16) out16[d] = ofe::from_float<T>(f);
        else out[d] = f;
    }
    return make_float2(m, l);
}

template <class T, int DP, int H>
__global__ void __launch_bounds__(Shape<DP, H>::kThreads, Shape<DP, H>::kBlocks) attention_kernel(const Args a, const __grid_constant__ CUtensorMap map_q,
                                                                                                  const __grid_constant__ CUtensorMap map_k,
                                                                                                  const __grid_constant__ CUtensorMap map_v,
                                                                                                  const __grid_constant__ CUtensorMap map_out) {
    using S = Shape<DP, H>;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    // ---- which rows, which keys.  The last rows come first: under a causal mask they have the most keys.
    const int split = blockIdx.x % a.splits, rest = blockIdx.x / a.splits;
    const int pairs = a.kv_heads * a.sequences;
    const int kh = rest % pairs % a.kv_heads, seq = rest % pairs / a.kv_heads, block = a.tiles - 1 - rest / pairs;
    int q0, nq, k0, nk;
    span(a.q_start, a.q_used, seq, a.q_rows, a.max_q, &q0, &nq);
    span(a.k_start, a.k_used, seq, a.k_rows, a.max_k, &k0, &nk);
    const int rows = nq * a.group, r0 = block * H * kRows;
    if (r0 >= rows) return;
    int lo[H], hi[H];  // the keys that a half's rows see between them
    int all_lo = 0, all_hi = 0;
#pragma unroll
    for (int x = 0; x < H; ++x) {
        int unused;
        lo[x] = hi[x] = 0;
        if (r0 + x * kRows >= rows) continue;
        window(a, a.by_group.quotient(r0 + x * kRows), nq, nk, &lo[x], &unused);
        window(a, a.by_group.quotient(min(r0 + (x + 1) * kRows, rows) - 1), nq, nk, &unused, &hi[x]);
        if (hi[x] <= lo[x]) continue;
        all_lo = all_hi == 0 ? lo[x] : min(all_lo, lo[x]);
        all_hi = max(all_hi, hi[x]);
    }
    const int tiles = (all_hi - all_lo + kKeys - 1) / kKeys, per = (tiles + a.splits - 1) / a.splits;
    const int first = min(split * per, tiles), count = min(per, tiles - first);  // this split's tiles
    const int base = all_lo + first * kKeys;                                     // and its first key
    int from[H], to[H];                                                          // each half's of them
#pragma unroll
    for (int x = 0; x < H; ++x) {
        from[x] = max((lo[x] - base) / kKeys, 0);  // (a negative difference rounds up: no further than 0)
        to[x] = hi[x] <= lo[x] ? 0 : min(max(hi[x] - base + kKeys - 1, 0) / kKeys, count);
        if (to[x] <= from[x]) from[x] = to[x] = 0;
    }

    extern __shared__ __align__(1024) uint8_t q_tiles[];  // the swizzle counts from 1024-byte boundaries
    uint8_t *const ring = q_tiles + H * S::kQueryBytes;
    uint64_t *const full = reinterpret_cast<uint64_t *>(ring + S::kStages * S::kStageBytes), *const empty = full + S::kStages;
    uint64_t *const my_turn = empty + S::kStages, *const ended = my_turn + H, *const of_half = ended + H;
    uint32_t *const tmem_slot = reinterpret_cast<uint32_t *>(of_half + H * S::kHalfBarriers);
    volatile int *const given_up = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const auto load = [&](int step, int stage) {
        const bool keys = step < count, values = step >= S::kBuffers;
        uint8_t *const at = ring + stage * S::kStageBytes;
        ofd::mbar_arrive_expect_tx(&full[stage], ((int)keys + (int)values) * S::kTileBytes);
#pragma unroll
        for (int d = 0; d < S::kChunks; ++d) {
            if (keys) tc5::load_3d(at + d * kKeys * 128, &map_k, d * 64, kh, k0 + base + step * kKeys, &full[stage]);
            if (values) tc5::load_3d(at + S::kTileBytes + d * kKeys * 128, &map_v, d * 64, kh, k0 + base + (step - S::kBuffers) * kKeys, &full[stage]);
        }
    };
    const int steps = count > 0 ? count + S::kBuffers : 0;
    if (threadIdx.x == 0) {
        *given_up = 0;
        for (int i = 0; i < S::kStages; ++i) {
            ofd::mbar_init(&full[i], 1);
            ofd::mbar_init(&empty[i], H);
        }
        for (int i = 0; i < 2 * H; ++i) ofd::mbar_init(&my_turn[i], 1);  // (and `ended`)
        for (int i = 0; i < H * S::kHalfBarriers; ++i) {
            // s_full and o_done are a commit's, p_ready takes an arrival of each warp, and so does q_ready without a copy
            const int of = i % S::kHalfBarriers;
            ofd::mbar_init(&of_half[i], of < S::kBuffers || of > 2 * S::kBuffers || (of == 2 * S::kBuffers && a.q_by_copy) ? 1 : 4);
        }
        ofd::mbar_fence_init();
        if (a.q_by_copy) {
            // rows that are not there come as whatever lies behind the sequence: each row of a product is by itself
#pragma unroll
            for (int i = 0; i < H; ++i) {
                if (to[i] <= from[i]) continue;
                uint64_t *const bar = of_half + i * S::kHalfBarriers + 2 * S::kBuffers;
                ofd::mbar_arrive_expect_tx(bar, S::kQueryBytes);
#pragma unroll
                for (int d = 0; d < S::kChunks; ++d)
                    tc5::load_3d(q_tiles + i * S::kQueryBytes + d * kRows * 128, &map_q, d * 64, kh * a.group,
                                 q0 + a.by_group.quotient(r0 + i * kRows), bar);
            }
        }
        for (int i = 0; i < S::kStages && i < steps; ++i) load(i, i);
    }
    if (warp == 4 * H) tc5::tmem_alloc<1>(tmem_slot, S::kColumns);
    tc5::before_sync();
    __syncthreads();
    tc5::after_sync();
    const int x = warp < 4 * H ? warp >> 2 : warp - 4 * H;  // this warp's half
    uint64_t *const s_full = of_half + x * S::kHalfBarriers, *const p_ready = s_full + S::kBuffers, *const q_ready = p_ready + S::kBuffers;
    uint64_t *const o_done = q_ready + 1;
    const uint32_t tmem = *tmem_slot + x * S::kHalfColumns;
    uint8_t *const q_tile = q_tiles + x * S::kQueryBytes;

    if (warp == 5 * H) {
        if (lane == 0) {
            int stage = 0;
            uint32_t turn = 0;
            for (int step = S::kStages; step < steps; ++step) {
                if (!tc5::wait(&empty[stage], turn, given_up, &g_status)) break;
                load(step, stage);
                if (++stage == S::kStages) stage = 0, turn ^= 1;
            }
        }
    } else if (warp >= 4 * H) {
        // The instructions are issued one after the other by one thread, whose own pace counts: descriptors are sums with
        // constants, loops are unrolled, and O += P V of one tile and S of the next are one run of instructions.
        constexpr bool bf16 = __is_same(T, __nv_bfloat16);
        constexpr uint32_t idesc_s = tc5::idesc_f16(128, kKeys, bf16, false), idesc_o = tc5::idesc_f16(128, DP, bf16, true);
        const uint64_t q_desc = tc5::desc_k_major(tc5::smem_u32(q_tile));
        const int begin = H == 1 ? 0 : from[x], end = H == 1 ? count : to[x];
        bool fine = end <= begin || tc5::wait_warp(q_ready, 0, given_up, &g_status);
        int stage = 0;
        uint32_t turn = 0;
        for (int step = 0; step < steps && fine; ++step) {
            // S of tile `step`, the half's tile `i`; O += P V of the one that had its place before
            const int i = step - begin, buffer = i & (S::kBuffers - 1);
            const bool scores = H == 1 ? step < count : step >= begin && step < end;
            const bool sums = H == 1 ? step >= S::kBuffers : i >= S::kBuffers && step < end + S::kBuffers;
            const uint32_t s_at = tmem + buffer * kKeys, o_at = tmem + S::kOut;
            const uint64_t kd = tc5::desc_k_major(tc5::smem_u32(ring + stage * S::kStageBytes));
            const uint64_t vd = tc5::desc_mn_major(tc5::smem_u32(ring + stage * S::kStageBytes + S::kTileBytes), kKeys * 128);
            const int valid = min(nk - (base + (step - S::kBuffers) * kKeys), kKeys), pieces = (valid + 15) / 16;  // of 16 keys
            fine = tc5::wait_warp(&full[stage], turn, given_up, &g_status);
            if (sums) {
                if (fine && (valid & 15)) {
                    // rows behind the sequence's last key that the last piece takes in: weights of zero, times what is there
                    const int behind = 16 - (valid & 15);
                    for (int n = lane; n < behind * 8 * S::kChunks; n += 32) {
                        const int d = n / (behind * 8), in = n % (behind * 8);
                        *reinterpret_cast<uint4 *>(ring + stage * S::kStageBytes + S::kTileBytes + d * kKeys * 128 + valid * 128 + in * 16) =
                            make_uint4(0, 0, 0, 0);
                    }
                    tc5::fence_async();
                    __syncwarp();
                }
                fine = fine && tc5::wait_warp(&p_ready[buffer], (i - S::kBuffers) / S::kBuffers & 1, given_up, &g_status);
            }
            // The halves take turns, so that one's weights are worked out beside the other's products: both at once end
            // together, and then the matrix unit has nothing to do.
            if (H == 2) fine = fine && tc5::wait_warp(&my_turn[x], (step + x + 1) & 1, given_up, &g_status);
            tc5::after_sync();
            if (fine && tc5::elect()) {
                if (sums) {
                    const bool more = i > S::kBuffers;
                    if (pieces == 4) {
#pragma unroll
                        for (int n = 0; n < 4; ++n) tc5::mma_f16_tmem(o_at, s_at + n * 8, vd + n * (2048 >> 4), idesc_o, more || n > 0);
                    } else {
                        for (int n = 0; n < pieces; ++n) tc5::mma_f16_tmem(o_at, s_at + n * 8, vd + n * (2048 >> 4), idesc_o, more || n > 0);
                    }
                }
                if (scores) {
#pragma unroll
                    for (int n = 0; n < DP / 16; ++n)
                        tc5::mma_f16(s_at, q_desc + ((n >> 2) * (kRows * 128 >> 4) + (n & 3) * 2), kd + ((n >> 2) * (kKeys * 128 >> 4) + (n & 3) * 2), idesc_s, n > 0);
                    tc5::commit(&s_full[buffer]);
                } else if (sums) {
                    tc5::commit(&o_done[step - end]);  // the last ones, which no S follows
                }
                if (H == 2) tc5::arrive(&my_turn[x ^ 1]);
                if (S::kCopyWarp) tc5::commit(&empty[stage]);
                // The weights were there, so S before them was: the products of the last step are done.
                else if (step > 0 && step + S::kStages - 1 < steps) load(step + S::kStages - 1, stage == 0 ? S::kStages - 1 : stage - 1);
            }
            __syncwarp();
            if (++stage == S::kStages) stage = 0, turn ^= 1;
        }
    } else {
        const int begin = H == 1 ? 0 : from[x], end = H == 1 ? count : to[x];
        const int row = (warp & 3) * 32 + lane, half0 = r0 + x * kRows;  // of the half, and lane of tensor memory; the half's first
        const int r = half0 + row, i = a.by_group.quotient(r), head = kh * a.group + r - i * a.group;
        const bool there = r < rows, warp_there = half0 + (warp & 3) * 32 < rows;
        // ---- the queries into shared memory, pieces of 16 bytes; zeros where there are none
        if (end > begin && !a.q_by_copy) {
            constexpr int kPieces = DP / 8;
#pragma unroll 4
            for (int n = threadIdx.x & 127; n < kRows * kPieces; n += 128) {
                const int qr = n / kPieces, p = n % kPieces, rr = half0 + qr, ri = a.by_group.quotient(rr);
                uint4 val = make_uint4(0, 0, 0, 0);
                if (rr < rows && p * 8 < a.head_dim)
                    val = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + (long long)(q0 + ri) * a.q_stride_row +
                                                           (kh * a.group + rr - ri * a.group) * a.q_stride_head + p * 8);
                *reinterpret_cast<uint4 *>(q_tile + (p >> 3) * kRows * 128 + qr * 128 + (((p & 7) ^ (qr & 7)) << 4)) = val;
            }
            tc5::fence_async();
            __syncwarp();
            if (lane == 0) tc5::arrive(q_ready);
        }
        // ---- the keys this row sees, none if it is not there, and between them the first and the last row of the warp that are
        int my_lo, my_hi;
        window(a, a.by_group.quotient(min(r, rows - 1)), nq, nk, &my_lo, &my_hi);
        const int first_lo = __shfl_sync(0xffffffffu, my_lo, 0), first_hi = __shfl_sync(0xffffffffu, my_hi, 0);
        const int last_lo = __shfl_sync(0xffffffffu, my_lo, 31), last_hi = __shfl_sync(0xffffffffu, my_hi, 31);
        if (!there) my_lo = my_hi = 0;
        float m = -INFINITY, l = 0.f;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, o_at = tmem + lanes + S::kOut;
        bool fine = true;
        for (int t = begin; t < end; ++t) {
            const int u = t - begin, buffer = u % S::kBuffers;
            fine = tc5::wait_warp(&s_full[buffer], u / S::kBuffers & 1, given_up, &g_status);
            if (!fine) break;
            tc5::after_sync();
            if (warp_there) {  // (else nothing but rows that are not there: their weights are whatever lies in the place)
                const uint32_t s_at = tmem + lanes + buffer * kKeys;
                const int j0 = base + t * kKeys;
                // In a tile that every row sees all of, the weights are worked out with the maximum there was before.  It is good
                // enough while their sum is below 2^15: then so is each of them, which every type can hold.
                bool careful = u == 0 || last_lo > j0 || first_hi < j0 + kKeys;
                if (!careful) {
                    uint32_t s[2][32], p[2][16];
                    tc5::ld64(s[0], s[1], s_at);
                    const float shift = fmaf(-m, a.c, kRoom<T>);
                    float2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            p[n][e] = weights<T>(__uint_as_float(s[n][e * 2]), __uint_as_float(s[n][e * 2 + 1]), a.c, shift, sum[e & 1]);
                    sum[0] = add2(sum[0], sum[1]);
                    const float tile_sum = sum[0].x + sum[0].y;
                    careful = __any_sync(0xffffffffu, my_hi != 0 && !(tile_sum <= kMostOfTile));  // (nor if it is no number)
                    if (!careful) {
                        tc5::st16(s_at, p[0]);
                        tc5::st16(s_at + 16, p[1]);
                        l += tile_sum;
                    }
                }
                if (careful) {
                    uint32_t s[2][32];
                    tc5::ld64(s[0], s[1], s_at);
                    float most = -INFINITY;
                    bool none[2];
#pragma unroll
                    for (int n = 0; n < 2; ++n) {  // 32 keys at a time: seen by none of the rows or by some
                        const int b = j0 + n * 32;
                        none[n] = first_lo >= b + 32 || last_hi <= b;
                        if (none[n]) continue;
                        const int lo_n = max(my_lo - b, 0), hi_n = min(my_hi - b, 32);
                        const uint32_t keep = hi_n <= lo_n ? 0u : (0xffffffffu >> (32 - (hi_n - lo_n))) << lo_n;
                        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                        for (int c = 0; c < 32; ++c) {
                            if (!(keep >> c & 1)) s[n][c] = 0xff800000u;  // -infinity
                            top[c & 1] = fmaxf(top[c & 1], __uint_as_float(s[n][c]));
                        }
                        most = max3(most, top[0], top[1]);
                    }
                    float fade = 1.f;
                    if (most > m) {
                        if (m == -INFINITY) {
                            m = most;
                        } else if ((most - m) * a.c > kLazy) {
                            fade = ex2((m - most) * a.c);
                            m = most;
                        }
                    }
                    if (__any_sync(0xffffffffu, fade != 1.f)) {
                        // the sums so far: with one S they are there when it is
                        // (else they are when the next tile's S is, which is formed behind them)
                        if (S::kBuffers == 2) fine = t + 1 < end ? tc5::wait_warp(&s_full[buffer ^ 1], (u + 1) / 2 & 1, given_up, &g_status)
                                                                 : tc5::wait_warp(&o_done[0], 0, given_up, &g_status);
                        tc5::after_sync();
                        l *= fade;
#pragma unroll 1
                        for (int n = 0; n < DP; n += 16) {
                            uint32_t o[16];
                            tc5::ld16(o, o_at + n);
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * fade);
                            tc5::st16(o_at + n, o);
                        }
                    }
                    const float shift = m == -INFINITY ? 0.f : fmaf(-m, a.c, kRoom<T>);
                    float2 sum = {0.f, 0.f};
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        uint32_t p[16];
                        if (none[n]) {
#pragma unroll
                            for (int e = 0; e < 16; ++e) p[e] = 0;
                        } else {
#pragma unroll
                            for (int e = 0; e < 16; ++e) p[e] = weights<T>(__uint_as_float(s[n][e * 2]), __uint_as_float(s[n][e * 2 + 1]), a.c, shift, sum);
                        }
                        tc5::st16(s_at + n * 16, p);
                    }
                    l += sum.x + sum.y;
                }
                tc5::st_wait();
            }
            if (!fine) break;
            tc5::before_sync();
            __syncwarp();
            if (lane == 0) tc5::arrive(&p_ready[buffer]);
        }
        // ---- out = O / l
        const bool any = fine && end > begin;
        if (any) {
            fine = tc5::wait_warp(&o_done[S::kBuffers - 1], 0, given_up, &g_status);
            tc5::after_sync();
        }
        if (fine && warp_there) {
            const int in_lo = max(my_lo, base), in_hi = min(my_hi, base + count * kKeys);  // of this split
            const bool sees = there && in_hi > in_lo;
            const float back = sees ? 1.f / l : 0.f;
            const long long at = split * a.part_step + ((long long)seq * a.max_q + i) * a.q_heads + head;
            T *const out = static_cast<T *>(a.out) + (long long)(q0 + i) * a.out_stride_row + head * a.out_stride_head;
            float *const part = a.part + at * a.head_dim;
            bool bad = false;
            // A warp whose rows are all there puts them where its queries were, and a tiled copy takes them out; else each thread
            // writes its own.
            const bool by_copy = a.out_by_copy && a.splits == 1 && half0 + (warp & 3) * 32 + 32 <= rows;
            uint8_t *const staged = q_tile + (warp & 3) * 4096;
#pragma unroll 1
            for (int n = 0; n < DP; n += 32) {
                uint32_t o[32];
                __syncwarp();
                if (any) tc5::ld32(o, o_at + n);
                if (!there) continue;
#pragma unroll
                for (int e = 0; e < 32; e += 8) {
                    if (n + e >= a.head_dim) break;
                    float f[8];
#pragma unroll
                    for (int b = 0; b < 8; ++b) {
                        f[b] = sees ? __uint_as_float(o[e + b]) * back : 0.f;
                        bad |= !(fabsf(f[b]) <= kLargest<T>);
                    }
                    const uint4 packed = make_uint4(pack<T>(f[0], f[1]), pack<T>(f[2], f[3]), pack<T>(f[4], f[5]), pack<T>(f[6], f[7]));
                    if (by_copy) {
                        *reinterpret_cast<uint4 *>(staged + ((n + e) >> 6) * kRows * 128 + lane * 128 + ((((n + e) >> 3 & 7) ^ (lane & 7)) << 4)) = packed;
                    } else if (a.splits == 1) {
                        *reinterpret_cast<uint4 *>(out + n + e) = packed;
                    } else {
                        *reinterpret_cast<float4 *>(part + n + e) = make_float4(f[0], f[1], f[2], f[3]);
                        *reinterpret_cast<float4 *>(part + n + e + 4) = make_float4(f[4], f[5], f[6], f[7]);
                    }
                }
            }
            if (by_copy) {
                if (!__any_sync(0xffffffffu, bad)) {
                    tc5::fence_async();
                    __syncwarp();
                    if (lane == 0) {
                        const int first_row = half0 + (warp & 3) * 32, token = a.by_group.quotient(first_row);
#pragma unroll
                        for (int d = 0; d < S::kChunks; ++d)
                            if (d * 64 < a.head_dim)
                                tc5::store_3d(&map_out, d * 64, kh * a.group + first_row - token * a.group, q0 + token, staged + d * kRows * 128);
                        tc5::store_commit();
                        tc5::store_wait_read<0>();
                    }
                } else {  // (the rows that are done again must not meet a copy that is under way)
                    for (int n = 0; n < a.head_dim; n += 8)
                        *reinterpret_cast<uint4 *>(out + n) =
                            *reinterpret_cast<const uint4 *>(staged + (n >> 6) * kRows * 128 + lane * 128 + (((n >> 3 & 7) ^ (lane & 7)) << 4));
                }
            }
            float lse = sees ? m * a.c + (log2f(l) - kRoom<T>) : -INFINITY;
            __syncwarp();
            for (uint32_t again = __ballot_sync(0xffffffffu, bad); again; again &= again - 1) {
                const int who = __ffs(again) - 1;
                const int rr = half0 + (warp & 3) * 32 + who, ii = a.by_group.quotient(rr), hh = kh * a.group + rr - ii * a.group;
                const int klo = __shfl_sync(0xffffffffu, in_lo, who), khi = __shfl_sync(0xffffffffu, in_hi, who);
                const long long aa = split * a.part_step + ((long long)seq * a.max_q + ii) * a.q_heads + hh;
                const float2 ml = redo_row<T>(static_cast<const T *>(a.q) + (long long)(q0 + ii) * a.q_stride_row + hh * a.q_stride_head,
                                              static_cast<const T *>(a.k) + (long long)k0 * a.k_stride_row + kh * a.k_stride_head,
                                              static_cast<const T *>(a.v) + (long long)k0 * a.v_stride_row + kh * a.v_stride_head, a.k_stride_row,
                                              a.v_stride_row, a.head_dim, a.c, klo, khi,
                                              a.part + aa * a.head_dim,
                                              a.splits > 1 ? nullptr : static_cast<T *>(a.out) + (long long)(q0 + ii) * a.out_stride_row + hh * a.out_stride_head);
                if (lane == who) lse = ml.x * a.c + log2f(ml.y);
            }
            if (a.splits > 1 && there) a.part_lse[at] = lse;
        }
    }
    __syncwarp();
    tc5::before_sync();
    __syncthreads();
    tc5::after_sync();
    if (*given_up) {
        // A wait has run out, whichever it was: what is under way lands before the block ends and gives its memory back.
        if (threadIdx.x == 0) {
            for (int n = 0; n < H; ++n)
                if (a.q_by_copy && to[n] > from[n]) ofd::mbar_land(of_half + n * S::kHalfBarriers + 2 * S::kBuffers, 0, 0, ofd::kDefaultWaitLimitNs / 16);
            for (int n = 0; n < S::kStages; ++n) {
                const uint64_t since = ofd::mbar_land(&full[n], 0, 0, ofd::kDefaultWaitLimitNs / 16);
                ofd::mbar_land(&full[n], 1, since, ofd::kDefaultWaitLimitNs / 16);
            }
        } else if (warp >= 4 * H && warp < 5 * H && tc5::elect()) {  // (the thread that has issued the products)
            tc5::commit(&ended[x]);
            ofd::mbar_land(&ended[x], 0, 0, ofd::kDefaultWaitLimitNs);
        }
        __syncwarp();
        __syncthreads();
    }
    if (warp == 4 * H) tc5::tmem_free<1>(tmem, S::kColumns);
}

// A single token to a sequence, R heads to a key head, which all see the same keys: what counts is to read those once.  LK lanes
// have 16 bytes each of a key and of its value, a slot of that many lanes takes every (kSlots)th key and keeps a maximum, a sum and
// results of its own, in fp32; the slots are joined at the end.  kAhead keys and values are on the way to every lane.
template <int LK, int R>
struct FewShape {
    static constexpr int kWarps = 4, kThreads = 32 * kWarps, kInWarp = 32 / LK, kSlots = kWarps * kInWarp, kAhead = 4;
    static constexpr int kBlocks = R == 1 ? 7 : 5;  // to an SM, by their registers
};

template <class T, int LK, int R>
__global__ void __launch_bounds__(FewShape<LK, R>::kThreads, FewShape<LK, R>::kBlocks) attention_few_kernel(const Args a) {
    using S = FewShape<LK, R>;
    __shared__ float sums[S::kWarps][R][LK * 8], tops[S::kWarps][R], totals[S::kWarps][R];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slot = warp * S::kInWarp + lane / LK, at = lane % LK * 8;
    const int split = blockIdx.x % a.splits, pair = blockIdx.x / a.splits, kh = pair % a.kv_heads, seq = pair / a.kv_heads;
    int q0, nq, k0, nk, lo, hi;
    span(a.q_start, a.q_used, seq, a.q_rows, a.max_q, &q0, &nq);
    if (nq == 0) return;
    span(a.k_start, a.k_used, seq, a.k_rows, a.max_k, &k0, &nk);
    window(a, 0, nq, nk, &lo, &hi);
    const int tiles = (max(hi - lo, 0) + kKeys - 1) / kKeys, per = (tiles + a.splits - 1) / a.splits;
    const int first = lo + min(split * per, tiles) * kKeys, last = min(first + per * kKeys, hi);
    const bool mine = at < a.head_dim;

    float2 q[R][4], acc[R][4] = {};
    float m[R], l[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        uint4 w = make_uint4(0, 0, 0, 0);
        if (mine)
            w = *reinterpret_cast<const uint4 *>(static_cast<const T *>(a.q) + (long long)q0 * a.q_stride_row + (kh * R + r) * a.q_stride_head + at);
        q[r][0] = ofe::unpack<T>(w.x);
        q[r][1] = ofe::unpack<T>(w.y);
        q[r][2] = ofe::unpack<T>(w.z);
        q[r][3] = ofe::unpack<T>(w.w);
        m[r] = -INFINITY;
        l[r] = 0.f;
    }
    const T *const keys = static_cast<const T *>(a.k) + (long long)k0 * a.k_stride_row + kh * a.k_stride_head + at;
    const T *const values = static_cast<const T *>(a.v) + (long long)k0 * a.v_stride_row + kh * a.v_stride_head + at;
    for (int j0 = first; j0 < last; j0 += S::kSlots * S::kAhead) {
        uint4 kw[S::kAhead], vw[S::kAhead];
        float z[R][S::kAhead];
#pragma unroll
        for (int n = 0; n < S::kAhead; ++n) {
            const int j = j0 + n * S::kSlots + slot;
            kw[n] = vw[n] = make_uint4(0, 0, 0, 0);
            if (j < last && mine) {
                kw[n] = __ldcs(reinterpret_cast<const uint4 *>(keys + j * a.k_stride_row));
                vw[n] = __ldcs(reinterpret_cast<const uint4 *>(values + j * a.v_stride_row));
            }
        }
#pragma unroll
        for (int n = 0; n < S::kAhead; ++n) {
            const float2 f[4] = {ofe::unpack<T>(kw[n].x), ofe::unpack<T>(kw[n].y), ofe::unpack<T>(kw[n].z), ofe::unpack<T>(kw[n].w)};
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float2 dot = {0.f, 0.f};
#pragma unroll
                for (int e = 0; e < 4; ++e) dot = fma2(q[r][e], f[e], dot);
                z[r][n] = dot.x + dot.y;
            }
        }
#pragma unroll
        for (int d = LK / 2; d > 0; d >>= 1)
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int n = 0; n < S::kAhead; ++n) z[r][n] += __shfl_xor_sync(0xffffffffu, z[r][n], d);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            float top = m[r];
#pragma unroll
            for (int n = 0; n < S::kAhead; ++n) {
                if (j0 + n * S::kSlots + slot >= last) z[r][n] = -INFINITY;
                top = fmaxf(top, z[r][n]);
            }
            const float fade = m[r] == top ? 1.f : ex2((m[r] - top) * a.c), from = top == -INFINITY ? 0.f : top;
            m[r] = top;
            l[r] *= fade;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[r][e] = ofe::mul2(acc[r][e], {fade, fade});
#pragma unroll
            for (int n = 0; n < S::kAhead; ++n) {
                z[r][n] = ex2((z[r][n] - from) * a.c);
                l[r] += z[r][n];
            }
        }
#pragma unroll
        for (int n = 0; n < S::kAhead; ++n) {
            const float2 f[4] = {ofe::unpack<T>(vw[n].x), ofe::unpack<T>(vw[n].y), ofe::unpack<T>(vw[n].z), ofe::unpack<T>(vw[n].w)};
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[r][e] = fma2({z[r][n], z[r][n]}, f[e], acc[r][e]);
        }
    }
    // ---- the slots of a warp, then the warps
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float top = m[r];
#pragma unroll
        for (int d = LK; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        const float fade = m[r] == top ? 1.f : ex2((m[r] - top) * a.c);
        l[r] *= fade;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[r][e] = ofe::mul2(acc[r][e], {fade, fade});
#pragma unroll
        for (int d = LK; d < 32; d <<= 1) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], d);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                acc[r][e].x += __shfl_xor_sync(0xffffffffu, acc[r][e].x, d);
                acc[r][e].y += __shfl_xor_sync(0xffffffffu, acc[r][e].y, d);
            }
        }
        if (lane < LK) {
#pragma unroll
            for (int e = 0; e < 4; ++e) *reinterpret_cast<float2 *>(&sums[warp][r][at + e * 2]) = acc[r][e];
            if (lane == 0) {
                tops[warp][r] = top;
                totals[warp][r] = l[r];
            }
        }
    }
    __syncthreads();
    for (int n = threadIdx.x; n < R * a.head_dim; n += S::kThreads) {
        const int r = n / a.head_dim, d = n - r * a.head_dim, head = kh * R + r;
        float top = -INFINITY, total = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < S::kWarps; ++w) top = fmaxf(top, tops[w][r]);
#pragma unroll
        for (int w = 0; w < S::kWarps; ++w) {
            const float f = tops[w][r] == top ? 1.f : ex2((tops[w][r] - top) * a.c);
            total = fmaf(totals[w][r], f, total);
            sum = fmaf(sums[w][r][d], f, sum);
        }
        // (a sum that is no number makes every element none)
        const float o = last <= first ? 0.f : total == total ? sum / total : NAN;
        if (a.splits == 1) {
            static_cast<T *>(a.out)[(long long)q0 * a.out_stride_row + head * a.out_stride_head + d] = ofe::from_float<T>(o);
        } else {
            const long long to = split * a.part_step + (long long)seq * a.max_q * a.q_heads + head;
            a.part[to * a.head_dim + d] = o;
            if (d == 0) a.part_lse[to] = last <= first ? -INFINITY : top * a.c + log2f(total);
        }
    }
}

// The splits' results joined: out = sum_z 2^(lse_z - max) o_z / sum_z 2^(lse_z - max).  A block to a query and head, every
// fourth split to a warp; the sums are formed in the same order every time.
template <class T>
__global__ void __launch_bounds__(128) attention_join_kernel(const Args a) {
    __shared__ float sums[4][128];
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the splits are done, and what they wrote is there
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long per = (long long)a.max_q * a.q_heads, all = per * a.sequences;
    for (long long w = blockIdx.x; w < all; w += gridDim.x) {
        const int seq = (int)(w / per), i = (int)(w % per / a.q_heads), head = (int)(w % a.q_heads);
        int q0, nq, k0, nk, lo, hi;
        span(a.q_start, a.q_used, seq, a.q_rows, a.max_q, &q0, &nq);
        if (i >= nq) continue;
        span(a.k_start, a.k_used, seq, a.k_rows, a.max_k, &k0, &nk);
        window(a, i, nq, nk, &lo, &hi);
        const long long at = w, step = a.part_step;
        // a lane to two splits (there are at most 64); -infinity: nothing seen there, or nothing but -infinity
        float lse[2], top;
#pragma unroll
        for (int h = 0; h < 2; ++h) lse[h] = lane + 32 * h < a.splits ? a.part_lse[(lane + 32 * h) * step + at] : -INFINITY;
        top = fmaxf(lse[0], lse[1]);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        const float from = top == -INFINITY ? 0.f : top;
        const float f0 = ex2(lse[0] - from), f1 = ex2(lse[1] - from);
        float total = f0 + f1;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
        float acc[4] = {};
#pragma unroll 4
        for (int z = warp; z < a.splits; z += 4) {
            const float f = __shfl_sync(0xffffffffu, z < 32 ? f0 : f1, z & 31);
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                if (lane + 32 * n >= a.head_dim) continue;
                const float o = a.part[(z * step + at) * a.head_dim + lane + 32 * n];
                acc[n] = f == 0.f ? acc[n] : fmaf(f, o, acc[n]);  // (a split in which nothing was seen has no part)
            }
        }
#pragma unroll
        for (int n = 0; n < 4; ++n) sums[warp][lane + 32 * n] = acc[n];
        __syncthreads();
        const int d = threadIdx.x;
        if (d < a.head_dim) {
            const float sum = (sums[0][d] + sums[1][d]) + (sums[2][d] + sums[3][d]);
            static_cast<T *>(a.out)[(long long)(q0 + i) * a.out_stride_row + head * a.out_stride_head + d] = ofe::from_float<T>(hi > lo ? sum / total : 0.f);
        }
        __syncthreads();
    }
}

// Whether the calls' rows are few enough for attention_few_kernel: a token to a sequence, as many heads to a key head as its lanes have
// the instructions for.  By it and by the tiles, us: heads of 64, one, two, four to a key head, 256 sequences of 256 to 2048 keys 102 / 153,
// 119 / 183, 175 / 163, one of 4097 keys 8.4 / 12.7, 10.6 / 17.7, 11.1 / 13.1; heads of 128, one, two, four, 64 sequences of 1024 to 8192 keys
// 720 (6.6 TB/s) / 841, 243 / 206, 346 / 211.
bool few_for(const openfish_b200_attention_t *a) {
    const int group = a->q_heads / a->kv_heads;
    return a->max_q == 1 && (group == 1 || (group == 2 && a->head_dim <= 64));
}

// Halves to a block.
int halves_for(const openfish_b200_attention_t *a) { return a->head_dim > 64 && (long long)a->max_q * (a->q_heads / a->kv_heads) > kRows ? 2 : 1; }

// Into how many pieces a block's keys go: as many as fill the SMs, four tiles of keys to a piece at least.  Where a sequence's
// queries are one block (single tokens), what they wait for is the keys: two tiles to a piece (one token by 4097 keys, 8
// heads of 64 by the matrix instructions: 12.7 us, with four tiles 13.9); and where the SMs are nearly full as it is, three pieces of 16 tiles or more even
// out sequences of different lengths (one token each by 1024 to 8192 keys, 32 / 8 heads of 128, us by one, two, three, four pieces: 64
// sequences 246, 217, 214, 214, 32 sequences 195, 162, 143, 162; 64 of 8192 keys all 347, 355, 370, 373).  Four rounds over the SMs even
// themselves out (by one and three: 128 sequences 450, 450, 256 of 512 to 4096 keys 434, 480).
int splits_for(const openfish_b200_attention_t *a, int sms) {
    const long long group = a->q_heads / a->kv_heads, halves = halves_for(a), rows = halves * kRows;
    const long long room = (long long)sms * (few_for(a) ? (group == 1 ? FewShape<8, 1>::kBlocks : FewShape<8, 2>::kBlocks)
                                             : a->head_dim <= 64 ? Shape<64, 1>::kBlocks : Shape<128, 1>::kBlocks / halves);
    const long long blocks = (a->max_q * group + rows - 1) / rows * a->kv_heads * a->sequences;
    long long keys = a->max_k;
    if (a->window_left >= 0 && a->window_right >= 0) {
        const long long seen = (long long)a->window_left + a->window_right + 1 + rows / group;
        if (seen < keys) keys = seen;
    }
    const long long tiles = (keys + kKeys - 1) / kKeys;
    const bool one_block = a->max_q * group <= kRows;
    long long n = room / blocks;
    if (one_block && n < 4 && blocks < 4 * room) {
        const long long even = tiles / 16 < 3 ? tiles / 16 : 3;
        if (even > n) n = even;
    }
    if (n > tiles / (one_block ? 2 : 4)) n = tiles / (one_block ? 2 : 4);
    if (n > 64) n = 64;
    return n < 1 ? 1 : (int)n;
}

// [rows][heads][head_dim] in boxes of 64 elements, `box_heads` heads and `box_rows` rows.
bool heads_map(CUtensorMap *map, bool bf16, const void *base, int head_dim, int heads, long long rows, long long stride_row, long long stride_head,
               int box_heads, int box_rows) {
    const cuuint64_t dims[3] = {(cuuint64_t)head_dim, (cuuint64_t)heads, (cuuint64_t)rows};
    const cuuint64_t strides[2] = {(cuuint64_t)(heads > 1 ? stride_head : 128) * 2, (cuuint64_t)(rows > 1 ? stride_row : 128) * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows};
    return tc5::make_map(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, base, dims, strides, box);
}

template <class T>
int join(const Args &a, cudaStream_t stream) {
    if (a.splits == 1) return OPENFISH_B200_OK;
    const long long joins = (long long)a.max_q * a.q_heads * a.sequences;
    // its blocks come to the SMs while the last ones before them leave (one token by 4097 keys by the tiles: 14.8 us, without 15.4)
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(joins < 16384 ? joins : 16384));
    cfg.blockDim = dim3(128);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return ofe::cuda_status(cudaLaunchKernelEx(&cfg, attention_join_kernel<T>, a));
}

template <class T, int DP, int H>
int launch_tiles(const Args &a, const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv, const CUtensorMap &mo, cudaStream_t stream) {
    using S = Shape<DP, H>;
    const auto kernel = attention_kernel<T, DP, H>;
    if (const int rc = ofe::cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes))) return rc;
    const long long blocks = (long long)a.tiles * a.kv_heads * a.sequences * a.splits;
    kernel<<<(unsigned)blocks, S::kThreads, S::kBytes, stream>>>(a, mq, mk, mv, mo);
    if (const int rc = ofe::launched()) return rc;
    return join<T>(a, stream);
}

template <class T, int LK, int R>
int launch_few(const Args &a, cudaStream_t stream) {
    const long long blocks = (long long)a.kv_heads * a.sequences * a.splits;
    attention_few_kernel<T, LK, R><<<(unsigned)blocks, FewShape<LK, R>::kThreads, 0, stream>>>(a);
    if (const int rc = ofe::launched()) return rc;
    return join<T>(a, stream);
}
template <class T>
int run_few(const Args &a, cudaStream_t stream) {
    if (a.head_dim > 64) return launch_few<T, 16, 1>(a, stream);
    return a.group == 1 ? launch_few<T, 8, 1>(a, stream) : launch_few<T, 8, 2>(a, stream);
}

template <class T>
int launch_for(const openfish_b200_attention_t *p, const Args &a, const CUtensorMap &mq, const CUtensorMap &mk, const CUtensorMap &mv, const CUtensorMap &mo, int halves, cudaStream_t stream) {
    if (p->head_dim <= 64) return launch_tiles<T, 64, 1>(a, mq, mk, mv, mo, stream);
    return halves == 1 ? launch_tiles<T, 128, 1>(a, mq, mk, mv, mo, stream) : launch_tiles<T, 128, 2>(a, mq, mk, mv, mo, stream);
}

size_t part_bytes(const openfish_b200_attention_t *a, int splits) {
    return splits == 1 ? 0 : (size_t)splits * a->sequences * a->max_q * a->q_heads * (a->head_dim + 1) * sizeof(float);
}

}  // namespace

extern "C" size_t ofb_attention_workspace(const openfish_b200_attention_t *a) {
    int sms = 0;
    if (ofe::sm_count(&sms)) return 0;
    return part_bytes(a, splits_for(a, sms));
}

extern "C" int ofb_attention(void *stream, const openfish_b200_attention_t *p) {
    int sms = 0, device = 0;
    if (const int rc = ofe::sm_count(&sms, &device)) return rc;
    g_reports.begin(device, t_known);
    Args a;
    a.q_start = p->q_start; a.k_start = p->k_start; a.q_used = p->q_used; a.k_used = p->k_used;
    a.q = p->q; a.k = p->k; a.v = p->v; a.out = p->out;
    // a stride counts only where there is a second element along it
    a.q_stride_row = p->q_stride_row; a.q_stride_head = p->q_heads > 1 ? p->q_stride_head : 0;
    a.k_stride_row = p->k_stride_row; a.k_stride_head = p->kv_heads > 1 ? p->k_stride_head : 0;
    a.v_stride_row = p->v_stride_row; a.v_stride_head = p->kv_heads > 1 ? p->v_stride_head : 0;
    a.out_stride_row = p->out_stride_row; a.out_stride_head = p->q_heads > 1 ? p->out_stride_head : 0;
    a.q_rows = (int)p->q_rows; a.k_rows = (int)p->k_rows; a.q_heads = p->q_heads; a.kv_heads = p->kv_heads; a.group = p->q_heads / p->kv_heads;
    a.head_dim = p->head_dim; a.sequences = p->sequences; a.max_q = p->max_q; a.max_k = p->max_k;
    const int wide = 1 << 30;  // beyond any sequence
    a.left = p->window_left < wide ? p->window_left : -1;
    a.right = p->window_right < wide ? p->window_right : -1;
    a.by_group = ofe::Divider((uint32_t)a.group);
    a.c = p->scale * 1.4426950408889634f;
    const int halves = halves_for(p);
    a.tiles = (int)(((long long)p->max_q * a.group + halves * kRows - 1) / (halves * kRows));
    a.splits = splits_for(p, sms);
    a.part_step = (long long)p->sequences * p->max_q * p->q_heads;
    a.part_lse = static_cast<float *>(p->workspace);
    a.part = a.part_lse;
    if (a.splits > 1) {
        // sums first: their rows are read and written 16 bytes at a time
        a.part = static_cast<float *>(p->workspace);
        a.part_lse = a.part + a.splits * a.part_step * a.head_dim;
    }
    const bool bf16 = p->dtype == OPENFISH_B200_BF16;
    if (few_for(p)) return bf16 ? run_few<__nv_bfloat16>(a, (cudaStream_t)stream) : run_few<__half>(a, (cudaStream_t)stream);
    CUtensorMap mq, mk, mv, mo;
    const int d = p->head_dim, hk = p->kv_heads;
    bool made = p->k_rows == 0  // no keys at all: the kernel copies nothing, but a map has to be one of something
                    ? heads_map(&mk, bf16, p->q, d, 1, 1, 0, 0, 1, kKeys) && heads_map(&mv, bf16, p->q, d, 1, 1, 0, 0, 1, kKeys)
                    : heads_map(&mk, bf16, p->k, d, hk, p->k_rows, p->k_stride_row, p->k_stride_head, 1, kKeys) &&
                          heads_map(&mv, bf16, p->v, d, hk, p->k_rows, p->v_stride_row, p->v_stride_head, 1, kKeys);
    a.q_by_copy = kRows % a.group == 0;
    mq = mk;
    if (a.q_by_copy) made = made && heads_map(&mq, bf16, p->q, d, p->q_heads, p->q_rows, p->q_stride_row, p->q_stride_head, a.group, kRows / a.group);
    a.out_by_copy = 32 % a.group == 0;
    mo = mk;
    if (a.out_by_copy) made = made && heads_map(&mo, bf16, p->out, d, p->q_heads, p->q_rows, p->out_stride_row, p->out_stride_head, a.group, 32 / a.group);
    if (!made) return ofb_fail(OPENFISH_B200_ERR_CUDA, "the driver made no tensor map");
    return bf16 ? launch_for<__nv_bfloat16>(p, a, mq, mk, mv, mo, halves, (cudaStream_t)stream) : launch_for<__half>(p, a, mq, mk, mv, mo, halves, (cudaStream_t)stream);
}

extern "C" int ofb_attention_settle(void *stream, int *gave_up) { return ofe::settle((cudaStream_t)stream, g_status, g_reports, t_known, gave_up); }
extern "C" int ofb_attention_status(int **word) { return ofe::cuda_status(cudaGetSymbolAddress((void **)word, g_status)); }
