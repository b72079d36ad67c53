// matmul_i8.cu -- product of tokens and weights in 8-bit integers (openfish_b200_matmul_i8).
//
//   out[m][n] = x_scale[m] w_scale[n] sum_k x[m][k] w[n][k] + bias[n]
//
// A handful of tokens reads the weights once and is bound by that: matmul_few_kernel, four products to an
// instruction.  Anything else goes to the matrix instructions: matmul_tile_kernel.
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "encoder_device.cuh"
#include "tc5.cuh"

namespace {

__device__ int g_status;  // how many waits of the kernels have run out on this device
Reports g_reports;
thread_local int t_known[Reports::kDevices];

struct Args {
    const int8_t *x, *w;
    const float *x_scale, *w_scale;
    const void *bias;
    void *out;
    long long x_stride, w_stride, out_stride;
    int rows, cols, depth;
    bool by_copy;  // out goes through the tiled copies
};

// ---------------------------------------------------------------------------------------------------------------
// Tiles of 128 * CG tokens by BN channels.  CG = 2: a pair of blocks on two neighbouring SMs shares one tile, each holding half of
// the tokens and half of the channels' weights, so that a byte of shared memory is filled once and read by both.
// KS > 1: a cluster of KS blocks shares a tile, each with a slice of the depth; at the end each reads the others' sums of its rows.
//
// Warps: 0 issues the copies, 1 the matrix instructions, the ones from 4 on (a quarter of the accumulator's 128 lanes and half
// of its columns each) scale and store.  The accumulator is there twice, so that one tile's sums are stored while the next one's are
// formed; the scales of a tile are fetched while the last one is stored.
template <int CG, int BN>
struct Shape {
    static constexpr int kRowsB = BN / CG;                     // weights' rows in one block
    static constexpr int kStageBytes = (128 + kRowsB) * 128;   // 128 deep
    static constexpr int kParts = BN >= 128 ? 2 : 1, kPart = BN / kParts;  // of a tile's columns, each with its four warps
    static constexpr int kThreads = 128 + 128 * kParts;
    static constexpr int kStages = BN == 64 ? 7 : 5;
    static constexpr int kOutBytes = kParts * 4 * 4096;    // a warp's 32 rows of 64 results, twice
    static constexpr int kScaleBytes = kParts * 4 * kPart * 8; // a warp's channel scales and biases
    static constexpr int kBytes = 1024 + kStages * kStageBytes + kOutBytes + kScaleBytes + (2 * kStages + 5) * 8 + 16;
    static constexpr int kColumns = 2 * BN;                    // of tensor memory, a power of two
};

struct Walk {  // the tiles in the order in which they are taken: stripes of 8 tiles of tokens, through all channels each
    int tiles_m, tiles_n;
    ofe::Divider by_stripe, by_last;  // tiles of a stripe; tiles of tokens in the last one
    Walk(int m, int n) : tiles_m(m), tiles_n(n), by_stripe((uint32_t)n * 8u), by_last((uint32_t)((m - 1) % 8 + 1)) {}
    __device__ __forceinline__ void at(int t, int *m, int *n) const {
        const int stripe = by_stripe.quotient(t), in = t - stripe * 8 * tiles_n;
        if (stripe * 8 + 8 <= tiles_m) {
            *n = in >> 3;
            *m = stripe * 8 + (in & 7);
        } else {
            *n = by_last.quotient(in);
            *m = stripe * 8 + in - *n * (tiles_m - stripe * 8);
        }
    }
};

template <class T, int CG, int BN, int KS>
__global__ void __launch_bounds__(Shape<CG, BN>::kThreads, 1) matmul_tile_kernel(const Args a, const Walk walk, const __grid_constant__ CUtensorMap map_x,
                                                                                 const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_out) {
    using S = Shape<CG, BN>;
    extern __shared__ uint8_t raw[];
    uint8_t *const base = raw + ((1024 - (tc5::smem_u32(raw) & 1023)) & 1023);
    uint8_t *const out_stage = base + S::kStages * S::kStageBytes;
    float *const scale_stage = reinterpret_cast<float *>(out_stage + S::kOutBytes);
    uint64_t *const full = reinterpret_cast<uint64_t *>(out_stage + S::kOutBytes + S::kScaleBytes);
    uint64_t *const empty = full + S::kStages, *const sum_full = empty + S::kStages, *const sum_empty = sum_full + 2, *const done = sum_empty + 2;
    uint32_t *const tmem_slot = reinterpret_cast<uint32_t *>(done + 1);
    volatile int *const given_up = reinterpret_cast<volatile int *>(tmem_slot + 1), *const steps_issued = given_up + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = CG == 2 ? blockIdx.x & 1 : 0;
    const int slice = KS > 1 ? blockIdx.x % KS : 0;
    const int group = blockIdx.x / (CG * KS), groups = gridDim.x / (CG * KS);
    const int tiles = walk.tiles_m * walk.tiles_n;
    const int all_steps = (a.depth + 127) / 128, from = all_steps * slice / KS, steps = all_steps * (slice + 1) / KS;  // of the depth

    // With KS slices of the depth, each block of the cluster has every KSth row of the results: these rows, this column and the
    // seven behind it to a thread.
    constexpr int kMine = KS > 1 ? 128 / KS * 8 / S::kThreads + (KS > 4) : 1;
    float my_xs[kMine];
    float2 my_ws[4], my_bias[4];
    int my_row = 0, my_n = 0, tile_m = 0;
    if (KS > 1) {
        int tm, tn;
        walk.at(group, &tm, &tn);
        tile_m = tm * 128;
        my_row = threadIdx.x / 8 * KS + slice;
        my_n = tn * BN + threadIdx.x % 8 * 8;
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int row = tile_m + my_row + i * S::kThreads / 8 * KS;
            my_xs[i] = row < a.rows ? a.x_scale[row] : 0.f;
        }
        const T *const bias = static_cast<const T *>(a.bias);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float ws = my_n + e < a.cols ? a.w_scale[my_n + e] : 0.f, b = bias && my_n + e < a.cols ? ofe::to_float(bias[my_n + e]) : 0.f;
            if (e & 1) my_ws[e / 2].y = ws, my_bias[e / 2].y = b;
            else my_ws[e / 2].x = ws, my_bias[e / 2].x = b;
        }
    }
    if (threadIdx.x == 0) {
        *given_up = 0;
        for (int i = 0; i < S::kStages; ++i) {
            ofd::mbar_init(&full[i], 1);
            ofd::mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            ofd::mbar_init(&sum_full[i], 1);
            ofd::mbar_init(&sum_empty[i], 4 * S::kParts * CG);
        }
        ofd::mbar_init(done, 1);
        ofd::mbar_fence_init();
        tc5::prefetch_map(&map_x);
        tc5::prefetch_map(&map_w);
    }
    if (warp == 1) tc5::tmem_alloc<CG>(tmem_slot, S::kColumns);
    tc5::before_sync();
    __syncthreads();
    if (CG == 2) tc5::cluster_sync();
    tc5::after_sync();
    const uint32_t tmem = *tmem_slot;

    if (warp == 0) {
        // copies: each block its own rows; the bytes of both are counted at the first block's barrier
        int stage = 0, issued = 0;
        uint32_t turn = 0;
        bool fine = true;
        for (int t = group; t < tiles && fine; t += groups) {
            int tm, tn;
            walk.at(t, &tm, &tn);
            const int m = tm * 128 * CG + rank * 128, n = tn * BN + rank * S::kRowsB;
            for (int k = from; k < steps; ++k, ++issued) {
                fine = tc5::wait_warp(&empty[stage], turn ^ 1, given_up, &g_status);
                if (!fine) break;
                uint8_t *const to = base + stage * S::kStageBytes;
                if (tc5::elect()) {
                    if (CG == 1) {
                        ofd::mbar_arrive_expect_tx(&full[stage], S::kStageBytes);
                        tc5::load_2d(to, &map_x, k * 128, m, &full[stage]);
                        tc5::load_2d(to + 128 * 128, &map_w, k * 128, n, &full[stage]);
                    } else {
                        if (rank == 0) ofd::mbar_arrive_expect_tx(&full[stage], 2 * S::kStageBytes);
                        const uint32_t bar = tc5::of_first_block(tc5::smem_u32(&full[stage]));
                        tc5::load_2d_pair(to, &map_x, k * 128, m, bar);
                        tc5::load_2d_pair(to + 128 * 128, &map_w, k * 128, n, bar);
                    }
                }
                __syncwarp();
                if (++stage == S::kStages) stage = 0, turn ^= 1;
            }
        }
        if (lane == 0) *steps_issued = issued;
    } else if (warp == 1 && rank == 0) {
        constexpr uint32_t idesc = tc5::idesc_i8(128 * CG, BN);
        const uint64_t base_a = tc5::desc_k_major(tc5::smem_u32(base)), base_b = tc5::desc_k_major(tc5::smem_u32(base) + 128 * 128);
        int stage = 0, j = 0;
        uint32_t turn = 0;
        bool fine = true;
        for (int t = group; t < tiles && fine; t += groups, ++j) {
            const uint32_t sum = tmem + (j & 1) * BN;
            fine = tc5::wait_warp(&sum_empty[j & 1], ((j >> 1) & 1) ^ 1, given_up, &g_status);
            for (int k = from; k < steps && fine; ++k) {
                fine = tc5::wait_warp(&full[stage], turn, given_up, &g_status);
                tc5::after_sync();
                const uint64_t da = base_a + (uint32_t)(stage * (S::kStageBytes >> 4)), db = base_b + (uint32_t)(stage * (S::kStageBytes >> 4));
                if (fine && tc5::elect()) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) tc5::mma_i8<CG>(sum, da + 2 * q, db + 2 * q, idesc, k > from || q > 0);
                    if (CG == 1) tc5::commit(&empty[stage]);
                    else tc5::commit_pair(&empty[stage]);
                    if (k + 1 == steps) {
                        if (CG == 1) tc5::commit(&sum_full[j & 1]);
                        else tc5::commit_pair(&sum_full[j & 1]);
                    }
                }
                __syncwarp();
                if (++stage == S::kStages) stage = 0, turn ^= 1;
            }
        }
    } else if (warp >= 4) {
        const int quarter = warp & 3, part = (warp - 4) >> 2;
        uint8_t *const mine = out_stage + (warp - 4) * 4096;
        float *const scales = scale_stage + (warp - 4) * 2 * S::kPart, *const biases = scales + S::kPart;
        const T *const bias = static_cast<const T *>(a.bias);
        float2 next[S::kPart / 32];  // the next tile's scales and biases, a lane to a column
        float next_xs = 0.f;
        int next_m0 = 0, next_n0 = 0;
        const auto fetch = [&](int t) {
            int tm, tn;
            walk.at(t, &tm, &tn);
            next_m0 = tm * 128 * CG + rank * 128 + quarter * 32;
            next_n0 = tn * BN + part * S::kPart;
            next_xs = next_m0 + lane < a.rows ? a.x_scale[next_m0 + lane] : 0.f;
#pragma unroll
            for (int i = 0; i < S::kPart / 32; ++i) {
                const int n = next_n0 + i * 32 + lane;
                next[i].x = n < a.cols ? a.w_scale[n] : 0.f;
                next[i].y = bias && n < a.cols ? ofe::to_float(bias[n]) : 0.f;
            }
        };
        if (KS == 1) fetch(group);
        int j = 0;
        for (int t = group; t < tiles; t += groups, ++j) {
            const int m0 = next_m0, n0 = next_n0;
            const float xs = next_xs;
            if (KS == 1) {
                __syncwarp();  // the last tile's scales have been read
#pragma unroll
                for (int i = 0; i < S::kPart / 32; ++i) {
                    scales[i * 32 + lane] = next[i].x;
                    biases[i * 32 + lane] = next[i].y;
                }
                __syncwarp();
                if (t + groups < tiles) fetch(t + groups);
            }
            if (!tc5::wait_warp(&sum_full[j & 1], (j >> 1) & 1, given_up, &g_status)) break;
            tc5::after_sync();
#pragma unroll 1
            for (int c = 0; c < S::kPart; c += 64) {
                const uint32_t sum = tmem + ((uint32_t)(quarter * 32) << 16) + (j & 1) * BN + part * S::kPart + c;
                uint32_t v[2][32];
                tc5::ld64(v[0], v[1], sum);
                if (KS > 1) {
                    // a slice's sums, where its tiles were (all of them have been read)
#pragma unroll
                    for (int p = 0; p < 16; ++p)
                        *reinterpret_cast<uint4 *>(base + (quarter * 32 + lane) * 256 + ((p ^ (lane & 7)) << 4)) =
                            make_uint4(v[p >> 3][(p & 7) * 4], v[p >> 3][(p & 7) * 4 + 1], v[p >> 3][(p & 7) * 4 + 2], v[p >> 3][(p & 7) * 4 + 3]);
                    continue;
                }
                if (c + 64 >= S::kPart) {  // the accumulator has been read: the next tile's sums may go there
                    tc5::before_sync();
                    __syncwarp();
                    if (lane == 0) {
                        if (CG == 1) tc5::arrive(&sum_empty[j & 1]);
                        else tc5::arrive_cluster(tc5::of_first_block(tc5::smem_u32(&sum_empty[j & 1])));
                    }
                }
                if (lane == 0) tc5::store_wait_read<0>();  // the copy out of this half of the staging memory is done with it
                __syncwarp();
                uint8_t *const to = mine;
#pragma unroll
                for (int p = 0; p < 8; ++p) {  // eight results, two to an instruction
                    uint32_t o[4];
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {
                        const float4 sw = *reinterpret_cast<const float4 *>(scales + c + p * 8 + e * 2);
                        float4 b = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (bias) b = *reinterpret_cast<const float4 *>(biases + c + p * 8 + e * 2);
                        const uint32_t *const sum4 = &v[p >> 2][(p & 3) * 8 + e * 2];
                        const float2 lo = ofe::fma2(ofe::mul2(make_float2((float)(int)sum4[0], (float)(int)sum4[1]), {xs, xs}), {sw.x, sw.y}, {b.x, b.y});
                        const float2 hi = ofe::fma2(ofe::mul2(make_float2((float)(int)sum4[2], (float)(int)sum4[3]), {xs, xs}), {sw.z, sw.w}, {b.z, b.w});
                        o[e] = ofe::pack<T>(lo.x, lo.y);
                        o[e + 1] = ofe::pack<T>(hi.x, hi.y);
                    }
                    *reinterpret_cast<uint4 *>(to + lane * 128 + ((p ^ (lane & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
                }
                if (a.by_copy) {
                    tc5::fence_async();
                    __syncwarp();
                    if (lane == 0) {
                        if (n0 + c < a.cols && m0 < a.rows) tc5::store_2d(&map_out, n0 + c, m0, to);
                        tc5::store_commit();
                    }
                } else {
                    // Rows of out that start anywhere: a row to an instruction, two results to a lane; a row that starts off a 4-byte
                    // boundary takes two instructions.  (53312 x 1538 and 1537 x 512: 68 and 74 us, 1536 by tiled copies 46.)
                    __syncwarp();
                    const int n = n0 + c, high = min(32, a.rows - m0), wide = min(64, a.cols - n);
                    uint16_t *out = static_cast<uint16_t *>(a.out) + (long long)m0 * a.out_stride + n;
                    if (high == 32 && wide == 64) {
                        // (n and the tile's first row are even: which rows start in front of a boundary is the same in every tile)
                        const auto rows = [&](auto first_odd, auto alternate) {
#pragma unroll 1
                            for (int r0 = 0; r0 < 32; r0 += 8) {
                                uint32_t two[8];
#pragma unroll
                                for (int r = 0; r < 8; ++r) two[r] = *reinterpret_cast<const uint32_t *>(to + (r0 + r) * 128 + (((lane >> 2) ^ r) << 4) + (lane & 3) * 4);
#pragma unroll
                                for (int r = 0; r < 8; ++r, out += a.out_stride) {
                                    if (first_odd.value != (alternate.value && (r & 1))) {
                                        out[2 * lane] = (uint16_t)two[r];
                                        out[2 * lane + 1] = (uint16_t)(two[r] >> 16);
                                    } else {
                                        *reinterpret_cast<uint32_t *>(out + 2 * lane) = two[r];
                                    }
                                }
                            }
                        };
                        const bool odd = (uintptr_t)a.out & 2, alternate = a.out_stride & 1;
                        if (alternate) odd ? rows(std::true_type(), std::true_type()) : rows(std::false_type(), std::true_type());
                        else odd ? rows(std::true_type(), std::false_type()) : rows(std::false_type(), std::false_type());
                    } else {
                        for (int r = 0; r < high; ++r, out += a.out_stride) {
                            const uint32_t two = *reinterpret_cast<const uint32_t *>(to + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
                            if (2 * lane < wide) out[2 * lane] = (uint16_t)two;
                            if (2 * lane + 1 < wide) out[2 * lane + 1] = (uint16_t)(two >> 16);
                        }
                    }
                    __syncwarp();
                }
            }
        }
        if (lane == 0) tc5::store_wait_read<0>();
    }
    __syncwarp();
    if (CG == 2 && lane == 0 && *given_up) tc5::store_peer_word(given_up, rank ^ 1, 1);  // a pair gives up together
    __syncwarp();
    tc5::before_sync();
    __syncthreads();
    if (CG == 2 || KS > 1) tc5::cluster_sync();
    tc5::after_sync();
    if (*given_up) {
        // A wait has run out, whichever it was: what is under way lands before the block (or its pair) ends and gives its memory back.
        if (warp == 0 && rank == 0 && lane == 0) {
            const uint64_t since = ofd::global_timer_ns();
            land_copies(
                *steps_issued, CG == 2 ? tc5::load_peer_word(steps_issued, 1) : *steps_issued, S::kStages,
                [&](int stage) { ofd::mbar_arrive_expect_tx(&full[stage], S::kStageBytes); },
                [&](int stage) { tc5::complete_tx(&full[stage], S::kStageBytes); },
                [&](int stage, uint32_t parity) { ofd::mbar_land(&full[stage], parity, since, ofd::kDefaultWaitLimitNs); });
        } else if (warp == 1 && rank == 0) {
            if (tc5::elect()) {  // (the thread that has issued them)
                tc5::commit<CG>(done);
                ofd::mbar_land(done, 0, 0, ofd::kDefaultWaitLimitNs);
            }
        }
        __syncwarp();
        if (CG == 2) tc5::cluster_sync();
        else __syncthreads();
    }
    if (KS > 1) {
        const uint32_t at = tc5::smem_u32(base);
#pragma unroll
        for (int i = 0; i < kMine; ++i) {
            const int row = my_row + i * S::kThreads / 8 * KS;
            if (row >= 128 || tile_m + row >= a.rows) continue;
            const int c = threadIdx.x % 8 * 2;
            int4 lo = make_int4(0, 0, 0, 0), hi = lo;
#pragma unroll
            for (int z = 0; z < KS; ++z) {
                const int4 p = tc5::load_peer(at + row * 256 + ((c ^ (row & 7)) << 4), z), q = tc5::load_peer(at + row * 256 + (((c + 1) ^ (row & 7)) << 4), z);
                lo.x += p.x, lo.y += p.y, lo.z += p.z, lo.w += p.w;
                hi.x += q.x, hi.y += q.y, hi.z += q.z, hi.w += q.w;
            }
            const float2 sum[4] = {{(float)lo.x, (float)lo.y}, {(float)lo.z, (float)lo.w}, {(float)hi.x, (float)hi.y}, {(float)hi.z, (float)hi.w}};
            uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 f = ofe::fma2(ofe::mul2(sum[e], {my_xs[i], my_xs[i]}), my_ws[e], my_bias[e]);
                o[e] = ofe::pack<T>(f.x, f.y);
            }
            uint16_t *const out = static_cast<uint16_t *>(a.out) + (long long)(tile_m + row) * a.out_stride + my_n;
            if (a.by_copy && my_n + 8 <= a.cols) {
                *reinterpret_cast<uint4 *>(out) = make_uint4(o[0], o[1], o[2], o[3]);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (my_n + e < a.cols) out[e] = (uint16_t)(o[e / 2] >> (e & 1) * 16);
            }
        }
        __syncwarp();
        tc5::cluster_sync();  // a block's memory stays until the others have read it
    }
    if (warp == 1) tc5::tmem_free<CG>(tmem, S::kColumns);
}

template <class T, int CG, int BN, int KS = 1>
int launch_tiles(const Args &a, int sms, cudaStream_t stream) {
    using S = Shape<CG, BN>;
    CUtensorMap mx, mw, mo;
    const auto map8 = [](CUtensorMap *map, const int8_t *base, int rows, int depth, long long stride, int box_rows) {
        const cuuint64_t dims[2] = {(cuuint64_t)depth, (cuuint64_t)rows};
        const cuuint64_t strides[1] = {rows > 1 ? (cuuint64_t)stride : (cuuint64_t)((depth + 15) / 16 * 16)};
        const cuuint32_t box[2] = {128, (cuuint32_t)box_rows};
        return tc5::make_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box);
    };
    bool made = map8(&mx, a.x, a.rows, a.depth, a.x_stride, 128) && map8(&mw, a.w, a.cols, a.depth, a.w_stride, S::kRowsB);
    if (made && a.by_copy && KS == 1) {
        const cuuint64_t dims[2] = {(cuuint64_t)a.cols, (cuuint64_t)a.rows};
        const cuuint64_t strides[1] = {(cuuint64_t)(a.rows > 1 ? a.out_stride : (a.cols + 7) / 8 * 8) * 2};
        const cuuint32_t box[2] = {64, 32};
        made = tc5::make_map(&mo, sizeof(T) == 2 ? CU_TENSOR_MAP_DATA_TYPE_UINT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, a.out, dims, strides, box);
    } else {
        mo = mw;
    }
    if (!made) return ofb_fail(OPENFISH_B200_ERR_CUDA, "the driver made no tensor map");
    const auto kernel = matmul_tile_kernel<T, CG, BN, KS>;
    if (const int rc = ofe::cuda_status(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes))) return rc;
    const Walk walk((a.rows + 128 * CG - 1) / (128 * CG), (a.cols + BN - 1) / BN);
    const long long tiles = (long long)walk.tiles_m * walk.tiles_n;
    const int most = sms / CG;  // (with slices there is a cluster to every tile)
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((KS > 1 ? tiles * KS : (tiles < most ? tiles : most) * CG)));
    cfg.blockDim = dim3(S::kThreads);
    cfg.dynamicSmemBytes = S::kBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CG * KS;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = CG * KS > 1 ? 1 : 0;
    return ofe::cuda_status(cudaLaunchKernelEx(&cfg, kernel, a, walk, mx, mw, mo));
}

// ---------------------------------------------------------------------------------------------------------------
// A few tokens: a warp to a channel, its lanes 16 bytes of the weights at a time; the tokens come from the cache.
template <class T, int MT>
__global__ void __launch_bounds__(128) matmul_few_kernel(const Args a) {
    const int lane = threadIdx.x & 31;
    const int n = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (n >= a.cols) return;
    const int8_t *const w = a.w + (long long)n * a.w_stride;
    const int8_t *x[MT];  // (tokens that are not there: the last one again)
    int sum[MT] = {};
#pragma unroll
    for (int i = 0; i < MT; ++i) x[i] = a.x + min(i, a.rows - 1) * a.x_stride;
    const auto add = [&](int k, int keep) {  // 16 of the depth, `keep` of them in it
        int4 wv = *reinterpret_cast<const int4 *>(w + k), xv[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i) xv[i] = *reinterpret_cast<const int4 *>(x[i] + k);
        if (keep < 16) {
            int *const word = reinterpret_cast<int *>(&wv);
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                const int left = keep - 4 * b;  // bytes of this word
                word[b] = left >= 4 ? word[b] : left <= 0 ? 0 : word[b] & ((1 << (8 * left)) - 1);
            }
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            sum[i] = __dp4a(xv[i].x, wv.x, sum[i]);
            sum[i] = __dp4a(xv[i].y, wv.y, sum[i]);
            sum[i] = __dp4a(xv[i].z, wv.z, sum[i]);
            sum[i] = __dp4a(xv[i].w, wv.w, sum[i]);
        }
    };
    int k = lane * 16;
#pragma unroll 4
    for (; k + 16 <= a.depth; k += 512) add(k, 16);
    if (k < a.depth) add(k, a.depth - k);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int s = __reduce_add_sync(0xffffffffu, sum[i]);
        if (lane == i && i < a.rows) {
            const float b = a.bias ? ofe::to_float(static_cast<const T *>(a.bias)[n]) : 0.f;
            static_cast<T *>(a.out)[i * a.out_stride + n] = ofe::from_float<T>(fmaf((float)s * a.x_scale[i], a.w_scale[n], b));
        }
    }
}

template <class T, int MT>
int launch_few(const Args &a, cudaStream_t stream) {
    matmul_few_kernel<T, MT><<<(unsigned)((a.cols + 3) / 4), 128, 0, stream>>>(a);
    return ofe::launched();
}

// Up to 8 tokens go to the dot products: us for 1, 4 and 8 tokens there / by the smallest tiles, 4096 x 4096: 3.4, 4.8, 7.5 / 14; 8192 x 1024: 2.7,
// 4.5, 6.5 / 6.7; 512 x 512: 1.6, 2.1, 2.6 / 3.9.
// Of the tiles, those whose rounds over the SMs are estimated to end first: a start, and a time for every 128 of the depth of a
// round.  Measured (us by 64, 128, 256 wide tiles, the chosen one first): 512 x 1536 x 512 4.3, 4.8, 6.6; 512 x 8192 x 1024 8.0 (256), 8.5, 11.8; 1003 x 2504 x
// 1237 8.8 (256), 10.3, 11.0; 2048 x 1536 x 512 6.2 (128), 6.7, 6.8; 4096 x 4096 x 4096 45 (256), 62, 109.
// Where there are few tiles and much depth, a cluster of 2, 4 or 8 blocks takes a tile, a slice of the depth to each (sums of integers: exact
// in any order).  us by one, two, four, eight: 64 x 4096 x 4096 10.4, 8.2 (four do not fit); 64 x 1024 x 4096 10.5, 8.1, 6.6, 10.9 (eight blocks to 16 tiles do not
// all find a place, so half the SMs bound these); 64 x 512 x 2048 6.9, 6.2, 5.6, 5.4; 64 x 256 x 16384 32.3, 18.9, 11.9, 8.6; 64 x 512 x 512
// 4.1, 4.8, 4.9.
template <class T>
int run(const Args &a, int sms, cudaStream_t stream) {
    if (a.rows <= 1) return launch_few<T, 1>(a, stream);
    if (a.rows <= 2) return launch_few<T, 2>(a, stream);
    if (a.rows <= 4) return launch_few<T, 4>(a, stream);
    if (a.rows <= 8) return launch_few<T, 8>(a, stream);
    const auto estimate = [&](int high, int wide, int at_once, double start, double step) {
        const double tiles = (double)((a.rows + high - 1) / high) * ((a.cols + wide - 1) / wide);
        return start + ceil(tiles / at_once) * ((a.depth + 127) / 128) * step;
    };
    const double t64 = estimate(128, 64, sms, 3.0, 0.25), t128 = estimate(128, 128, sms, 3.6, 0.30), t256 = estimate(256, 256, sms / 2, 5.4, 0.36);
    const long long tiles = (long long)((a.rows + 127) / 128) * ((a.cols + 63) / 64);
    int slices = 1;
    double best = t64 < t128 ? t64 : t128;
    if (t256 < best) best = t256;
    const double joins[3] = {1.2, 1.6, 1.9};
    for (int i = 0; i < 3; ++i) {
        const int n = 2 << i, steps = (a.depth + 127) / 128;
        const double time = 3.0 + joins[i] + (steps + n - 1) / n * 0.25;
        if (tiles * n <= (n == 8 ? sms / 2 : sms) && steps >= n && time < best) {
            best = time;
            slices = n;
        }
    }
    if (slices == 2) return launch_tiles<T, 1, 64, 2>(a, sms, stream);
    if (slices == 4) return launch_tiles<T, 1, 64, 4>(a, sms, stream);
    if (slices == 8) return launch_tiles<T, 1, 64, 8>(a, sms, stream);
    if (t64 <= t128 && t64 <= t256) return launch_tiles<T, 1, 64>(a, sms, stream);
    return t128 < t256 ? launch_tiles<T, 1, 128>(a, sms, stream) : launch_tiles<T, 2, 256>(a, sms, stream);
}

}  // namespace

extern "C" int ofb_matmul_i8(void *stream, const openfish_b200_matmul_i8_t *p) {
    int sms = 0, device = 0;
    if (const int rc = ofe::sm_count(&sms, &device)) return rc;
    g_reports.begin(device, t_known);
    Args a;
    a.x = p->x; a.w = p->w; a.x_scale = p->x_scale; a.w_scale = p->w_scale; a.bias = p->bias; a.out = p->out;
    a.x_stride = p->x_stride; a.w_stride = p->w_stride; a.out_stride = p->out_stride;
    a.rows = (int)p->rows; a.cols = p->cols; a.depth = p->depth;
    a.by_copy = (uintptr_t)p->out % 16 == 0 && (p->rows == 1 || p->out_stride % 8 == 0);
    return p->dtype == OPENFISH_B200_F16 ? run<__half>(a, sms, (cudaStream_t)stream) : run<__nv_bfloat16>(a, sms, (cudaStream_t)stream);
}

extern "C" int ofb_matmul_i8_settle(void *stream, int *gave_up) { return ofe::settle((cudaStream_t)stream, g_status, g_reports, t_known, gave_up); }
extern "C" int ofb_matmul_i8_status(int **word) { return ofe::cuda_status(cudaGetSymbolAddress((void **)word, g_status)); }
