// Linear layers of many sub-networks over rows grouped by id: row i belongs to group g(i) and
//   y_i = act(W_g x_i + b_g),   dX_i = W_g^T dZ_i,   dW_g = sum_i dZ_i x_i^T,   db_g = sum_i dZ_i,   dZ = dY [y > 0].
// The reference has one network for all points (models/nerf.py:155-209); here the points of one call are dealt out to
// sub-networks (a spatial grid, a router), each with as many points as fall to it.
//
// Rows stay where they are: a tile is 128 consecutive positions of the grouped order, and the kernels read and write
// row order[position] of the ordinary tensors (a row is one or more whole cache lines, so gathering costs nothing).  The
// number of tiles is known on the device only: the grid is the upper bound n / 128 + groups + 1 and a workgroup finds its
// group in tile_base, the running number of tiles, with one or two 64-wide comparisons.
//
// Operands go through registers into LDS in 16-byte pieces, two buffers, one barrier per step; products run on
// v_mfma_f32_32x32x16_{bf16,f16} or, in fp32, v_mfma_f32_32x32x2_f32 (exact products, fp32 sums).  A 16-byte piece holds
// the values of consecutive contraction indices of one row; operands whose contraction index is the row (W in dX, both in
// dW) are read with ds_read_b64_tr_b16, which hands a lane four rows of its column, or in fp32 with four 4-byte reads.
// LDS pieces are permuted within a row so that the 16 (8) lanes of one LDS cycle fall on different banks.
#include "elems.hpp"
#include "groups.hpp"

namespace nerf {
namespace gl {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
using grp::TILE_ROWS;

constexpr int THREADS = 256;
constexpr int ROW_PIECES = 8;                     // 16-byte pieces of one contraction step in a row: 128 bytes
constexpr int MAX_CHUNK_TILES = 256;              // tiles one workgroup of the weight gradient walks

template <typename T> struct El;
template <> struct El<__bf16> {
    typedef __bf16 frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x16 mfma(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct El<_Float16> {
    typedef _Float16 frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x16 mfma(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct El<float> {
    // four contraction indices per lane: lanes 0-31 hold the first four of eight, lanes 32-63 the others, the same in
    // both operands
    typedef f32x4 frag;
    static __device__ __forceinline__ f32x16 mfma(frag a, frag b, f32x16 c) {
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
        return c;
    }
};

template <typename T> constexpr int piece() { return 16 / (int)sizeof(T); }             // elements of a piece
template <typename T> constexpr int step_len() { return ROW_PIECES * piece<T>(); }      // contraction indices of a step

// ---- row-major tile, contraction index within the row: [rows][8 pieces] ---------------------------------------
__device__ __forceinline__ int nt_addr(int row, int q) { return row * 128 + ((q ^ ((row >> 1) & 7)) << 4); }

template <typename T>
__device__ __forceinline__ typename El<T>::frag nt_frag(const char* tile, int row0, int s, int lane) {
    return *reinterpret_cast<const typename El<T>::frag*>(tile + nt_addr(row0 + (lane & 31), 2 * s + (lane >> 5)));
}

// ---- row-major tile, contraction index = row: [step_len rows][up to 128 columns] ------------------------------
template <typename T> constexpr int tr_pitch() { return sizeof(T) == 2 ? 256 : 544; }
template <typename T> constexpr int tr_bytes() { return step_len<T>() * tr_pitch<T>(); }
template <typename T>
__device__ __forceinline__ int tr_addr(int row, int q) {
    if constexpr (sizeof(T) == 2) return row * 256 + ((q ^ ((row & 3) << 2)) << 4);
    else return row * 544 + (q << 4);
}

template <typename T>
__device__ __forceinline__ typename El<T>::frag tr_frag(const char* tile, int col0, int s, int lane) {
    if constexpr (sizeof(T) == 2) {
        const int i = lane & 15;
        const int row = 16 * s + 8 * (lane >> 5) + (i >> 2);
        const int col = col0 + ((lane >> 4) & 1) * 16 + (i & 3) * 4;
        typedef __attribute__((address_space(3))) s16x4* lds_ptr;
        const int a = tr_addr<T>(row, col >> 3) + ((col >> 2) & 1) * 8;      // rows 4 apart share their permutation
        struct Two { s16x4 lo, hi; } f;
        f.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(tile + a));
        f.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(tile + a + 4 * 256));
        return __builtin_bit_cast(typename El<T>::frag, f);
    } else {
        const int row = 8 * s + 4 * (lane >> 5), col = col0 + (lane & 31);
        f32x4 f;
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = *reinterpret_cast<const float*>(tile + (row + j) * 544 + col * 4);
        return f;
    }
}

// ---- pieces from memory ---------------------------------------------------------------------------------------
// columns c .. of a row that has `cols` of them; zero behind its end and when !ok
template <typename T, bool WIDE>
__device__ __forceinline__ Pack<T, piece<T>()> load_piece(const T* row, int c, int cols, bool ok) {
    constexpr int E = piece<T>();
    Pack<T, E> p;
    if constexpr (WIDE) {
        if (ok && c < cols) return load_pack<T, E>(row + c);
#pragma unroll
        for (int e = 0; e < E; ++e) p.v[e] = (T)0.0f;
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) p.v[e] = ok && c + e < cols ? row[c + e] : (T)0.0f;
    }
    return p;
}

template <typename T, int E>
__device__ __forceinline__ void put_piece(char* at, const Pack<T, E>& p) { *reinterpret_cast<Pack<T, E>*>(at) = p; }

// gradient pieces where the layer's output was cut off by its ReLU become zero (a NaN output keeps its gradient)
template <typename T, int E>
__device__ __forceinline__ void gate_piece(Pack<T, E>& g, const Pack<T, E>& y) {
#pragma unroll
    for (int e = 0; e < E; ++e)
        if ((float)y.v[e] <= 0.0f) g.v[e] = (T)0.0f;
}

struct Rows {
    int64_t n;
    int n_groups;
    const int32_t *order, *offsets, *tile_base;
};

// row of a position; -1 for an entry that is no row
__device__ __forceinline__ int row_at(const Rows& r, int64_t pos) {
    if (!r.order) return (int)pos;
    const int row = r.order[pos];
    return row >= 0 && row < r.n ? row : -1;
}

struct LinArgs {
    Rows rows;
    int C, O, tiles_o;           // contraction length, outputs, output tiles
    int64_t a_ld;
    const void *a, *gate, *w, *bias;
    int relu;
    void* out;
};

// out[row][o] = sum_c a[row][c] w_g(o, c).  WT = false: w_g is [O][C] (the layer); WT = true: w_g is [C][O] (its data
// gradient).  A tile is 128 rows x BN outputs, four waves.  The accumulators hold outputs down and rows across, so a
// lane's four consecutive registers are consecutive outputs of one row.
template <typename T, bool WT, bool GATE, bool WIDE, int BN>
__global__ __launch_bounds__(THREADS, 2) void linear_kernel(LinArgs p) {
    constexpr int E = piece<T>(), BK = step_len<T>();
    constexpr int A_BYTES = TILE_ROWS * 128;
    constexpr int B_BYTES = WT ? tr_bytes<T>() : BN * 128;
    constexpr int STAGE = A_BYTES + B_BYTES;
    constexpr int PITCH = BN * 2 + 16;                                      // 16-bit output tile in LDS
    constexpr int LDS = 2 * STAGE > TILE_ROWS * PITCH ? 2 * STAGE : TILE_ROWS * PITCH;
    __shared__ __attribute__((aligned(16))) char lds[LDS];
    __shared__ int row_of[TILE_ROWS];
    constexpr int MI = BN == 128 ? 2 : 1, NJ = 2;                           // 32-row and 32-output tiles of a wave
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m_off = BN == 128 ? (wave & 1) * 64 : wave * 32, o_off = BN == 128 ? (wave >> 1) * 64 : 0;

    // consecutive tiles on one XCD (workgroups go round the eight XCDs), output tiles of the same rows next to each other
    const int G = p.rows.n_groups;
    const int64_t work = (int64_t)p.rows.tile_base[G + 1] * p.tiles_o;
    const int64_t per_xcd = (work + 7) / 8;
    const int64_t local = blockIdx.x >> 3;
    const int64_t at = (blockIdx.x & 7) * per_xcd + local;
    if (local >= per_xcd || at >= work) return;
    const int t = (int)(at / p.tiles_o), o0 = (int)(at % p.tiles_o) * BN;
    const int g = grp::group_of_tile(p.rows.tile_base, G, t, lane);
    const int64_t pos0 = p.rows.offsets[g] + (int64_t)(t - p.rows.tile_base[g]) * TILE_ROWS;
    const int64_t end = g < G ? (int64_t)p.rows.offsets[g + 1] : p.rows.n;
    const int count = (int)(end - pos0 < TILE_ROWS ? end - pos0 : TILE_ROWS);
    if (tid < TILE_ROWS) row_of[tid] = tid < count ? row_at(p.rows, pos0 + tid) : -1;
    __syncthreads();
    T* out = (T*)p.out;
    const int O = p.O, C = p.C;
    if (g == G) {                                                           // rows of no group
        const int width = O - o0 < BN ? O - o0 : BN;
        for (int i = tid; i < count * width; i += THREADS) {
            const int row = row_of[i / width];
            if (row >= 0) out[(int64_t)row * O + o0 + i % width] = (T)0.0f;
        }
        return;
    }

    const T* w = (const T*)p.w + (int64_t)g * O * C;
    // pieces of this thread: rows tid / 8 + 32 i of A (and of W), piece tid % 8
    const int q = tid & 7, r0 = tid >> 3;
    const T *arow[4], *yrow[4];
    bool aok[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int row = row_of[r0 + 32 * i];
        aok[i] = row >= 0;
        arow[i] = (const T*)p.a + (int64_t)(row < 0 ? 0 : row) * p.a_ld;
        if (GATE) yrow[i] = (const T*)p.gate + (int64_t)(row < 0 ? 0 : row) * C;
    }
    constexpr int BPR = BN / E;                                             // pieces per row of a transposed W tile
    constexpr int NB = WT ? BK * BPR / THREADS : BN / 32;
    Pack<T, E> ra[4], rb[NB];
    auto load = [&](int k0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            ra[i] = load_piece<T, WIDE>(arow[i], k0 + q * E, C, aok[i]);
            if (GATE) {
                const Pack<T, E> y = load_piece<T, WIDE>(yrow[i], k0 + q * E, C, aok[i]);
                gate_piece<T, E>(ra[i], y);
            }
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            if constexpr (WT) {
                const int c = k0 + tid / BPR + (THREADS / BPR) * i;
                rb[i] = load_piece<T, WIDE>(w + (int64_t)c * O, o0 + (tid % BPR) * E, O, c < C);
            } else {
                const int o = o0 + r0 + 32 * i;
                rb[i] = load_piece<T, WIDE>(w + (int64_t)o * C, k0 + q * E, C, o < O);
            }
        }
    };
    auto put = [&](int buf) {
        char* A = lds + buf * STAGE;
        char* B = A + A_BYTES;
#pragma unroll
        for (int i = 0; i < 4; ++i) put_piece<T, E>(A + nt_addr(r0 + 32 * i, q), ra[i]);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            if constexpr (WT) put_piece<T, E>(B + tr_addr<T>(tid / BPR + (THREADS / BPR) * i, tid % BPR), rb[i]);
            else put_piece<T, E>(B + nt_addr(r0 + 32 * i, q), rb[i]);
        }
    };

    f32x16 acc[MI][NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
        f32x16 b0;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int o = o0 + o_off + 32 * j + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
            b0[r] = p.bias && o < O ? (float)((const T*)p.bias)[(int64_t)g * O + o] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < MI; ++i) acc[i][j] = b0;
    }
    const int steps = (C + BK - 1) / BK;
    load(0);
    put(0);
    __syncthreads();
    for (int k = 0; k < steps; ++k) {
        if (k + 1 < steps) load((k + 1) * BK);
        const char* A = lds + (k & 1) * STAGE;
        const char* B = A + A_BYTES;
#pragma unroll
        for (int s = 0; s < ROW_PIECES / 2; ++s) {
            typename El<T>::frag fx[MI], fw[NJ];
#pragma unroll
            for (int i = 0; i < MI; ++i) fx[i] = nt_frag<T>(A, m_off + 32 * i, s, lane);
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                if constexpr (WT) fw[j] = tr_frag<T>(B, o_off + 32 * j, s, lane);
                else fw[j] = nt_frag<T>(B, o_off + 32 * j, s, lane);
            }
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NJ; ++j) acc[i][j] = El<T>::mfma(fw[j], fx[i], acc[i][j]);
        }
        if (k + 1 < steps) put((k + 1) & 1);
        __syncthreads();
    }
    if (p.relu) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = acc[i][j][r] < 0.0f ? 0.0f : acc[i][j][r];   // keeps a NaN
    }
    if constexpr (sizeof(T) == 2) {
        // through LDS, so that rows leave in 16-byte pieces of whole lines
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    Pack<T, 4> v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v.v[e] = (T)acc[i][j][4 * h + e];
                    put_piece<T, 4>(lds + (m_off + 32 * i + (lane & 31)) * PITCH + (o_off + 32 * j + 8 * h + 4 * (lane >> 5)) * 2, v);
                }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TILE_ROWS * BN / E / THREADS; ++i) {
            const int at2 = tid + i * THREADS, m = at2 / (BN / E), c = (at2 % (BN / E)) * E;
            const int row = row_of[m];
            if (row < 0 || o0 + c >= O) continue;
            const Pack<T, E> v = *reinterpret_cast<const Pack<T, E>*>(lds + m * PITCH + c * 2);
            T* to = out + (int64_t)row * O + o0 + c;
            if constexpr (WIDE) store_pack<T, E>(to, v);
            else
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (o0 + c + e < O) to[e] = v.v[e];
        }
    } else {
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            const int row = row_of[m_off + 32 * i + (lane & 31)];
            if (row < 0) continue;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const int o = o0 + o_off + 32 * j + 8 * h + 4 * (lane >> 5);
                    T* to = out + (int64_t)row * O + o;
                    if constexpr (WIDE) {
                        if (o < O) store_pack<float, 4>((float*)to, Pack<float, 4>{{acc[i][j][4 * h], acc[i][j][4 * h + 1], acc[i][j][4 * h + 2], acc[i][j][4 * h + 3]}});
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (o + e < O) to[e] = (T)acc[i][j][4 * h + e];
                    }
                }
        }
    }
}

struct WgradArgs {
    Rows rows;
    int K, N, tiles_k, tiles_n;
    int chunk;                       // tiles of one workgroup
    int64_t x_ld, dy_ld;
    const void *x, *dy, *y;
    void *dw, *db;
    float *part_w, *part_b;          // [2 * chunks][N * K], [2 * chunks][N]: slot 2c a group that came in from the left of
};                                   // chunk c, slot 2c + 1 one that began in it and goes on to the right

// dW[n][k] = sum over rows dZ[row][n] x[row][k].  A workgroup owns one BT x BT block of every dW it meets and walks
// `chunk` consecutive tiles of the flat tile list, whatever groups they belong to, so all workgroups have equal work
// however uneven the groups are.  A group that lies inside one chunk is finished here; the pieces of a longer one go to
// the workspace and are added up in order by wgrad_join_kernel (no atomics: the result does not depend on timing).
template <typename T, bool GATE, bool WIDE, int BT>
__global__ __launch_bounds__(THREADS, 2) void wgrad_kernel(WgradArgs p) {
    constexpr int E = piece<T>(), BK = step_len<T>();                       // rows of one step
    constexpr int PER_TILE = TILE_ROWS / BK;
    constexpr int STAGE = 2 * tr_bytes<T>();
    __shared__ __attribute__((aligned(16))) char lds[2 * STAGE];
    __shared__ int tile_pos[MAX_CHUNK_TILES], tile_cnt[MAX_CHUNK_TILES], tile_grp[MAX_CHUNK_TILES];
    constexpr int M = BT / 64;                                              // 32 x 32 blocks of a wave: M x M
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n_off = (wave & 1) * (BT / 2), k_off = (wave >> 1) * (BT / 2);

    // the blocks of one chunk next to each other on one XCD: they read the same rows
    const int G = p.rows.n_groups;
    const int tiles = p.rows.tile_base[G];                                  // the rows of no group stay out
    const int blocks = p.tiles_n * p.tiles_k;
    const int64_t work = (int64_t)((tiles + p.chunk - 1) / p.chunk) * blocks;
    const int64_t per_xcd = ((work + blocks - 1) / blocks + 7) / 8 * blocks;
    const int64_t local = blockIdx.x >> 3;
    const int64_t at = (blockIdx.x & 7) * per_xcd + local;
    if (local >= per_xcd || at >= work) return;
    const int c = (int)(at / blocks), blk = (int)(at % blocks);
    const int n0 = (blk / p.tiles_k) * BT, k0 = (blk % p.tiles_k) * BT;
    const int t0 = c * p.chunk, t1 = t0 + p.chunk < tiles ? t0 + p.chunk : tiles;
    for (int i = tid; i < t1 - t0; i += THREADS) {
        int lo = 0, hi = G;                                                 // last group with tile_base <= t
        const int t = t0 + i;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (p.rows.tile_base[mid] <= t) lo = mid;
            else hi = mid;
        }
        const int64_t pos = p.rows.offsets[lo] + (int64_t)(t - p.rows.tile_base[lo]) * TILE_ROWS;
        const int64_t left = p.rows.offsets[lo + 1] - pos;
        tile_pos[i] = (int)pos;
        tile_cnt[i] = (int)(left < TILE_ROWS ? left : TILE_ROWS);
        tile_grp[i] = lo;
    }
    __syncthreads();

    const int K = p.K, N = p.N;
    constexpr int BPR = BT / E, RSTEP = THREADS / BPR, NP = BK / RSTEP;     // pieces of a row, rows between a thread's pieces
    const int q = tid % BPR, r0 = tid / BPR;
    Pack<T, E> rx[NP], rd[NP];
    int rows[NP];
    const int steps = (t1 - t0) * PER_TILE;
    auto find = [&](int s) {                                                // rows of step s
        const int i = s / PER_TILE, first = (s % PER_TILE) * BK;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int r = first + r0 + RSTEP * j;
            rows[j] = s < steps && r < tile_cnt[i < t1 - t0 ? i : 0] ? row_at(p.rows, (int64_t)tile_pos[i] + r) : -1;
        }
    };
    auto load = [&]() {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const bool ok = rows[j] >= 0;
            const int64_t row = ok ? rows[j] : 0;
            rx[j] = load_piece<T, WIDE>((const T*)p.x + row * p.x_ld, k0 + q * E, K, ok);
            rd[j] = load_piece<T, WIDE>((const T*)p.dy + row * p.dy_ld, n0 + q * E, N, ok);
            if (GATE) {
                const Pack<T, E> y = load_piece<T, WIDE>((const T*)p.y + row * N, n0 + q * E, N, ok);
                gate_piece<T, E>(rd[j], y);
            }
        }
    };
    auto put = [&](int buf) {
        char* X = lds + buf * STAGE;
        char* D = X + tr_bytes<T>();
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            put_piece<T, E>(X + tr_addr<T>(r0 + RSTEP * j, q), rx[j]);
            put_piece<T, E>(D + tr_addr<T>(r0 + RSTEP * j, q), rd[j]);
        }
    };
    f32x16 acc[M][M], accb[M];
    auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < M; ++i) {
#pragma unroll
            for (int r = 0; r < 16; ++r) accb[i][r] = 0.0f;
#pragma unroll
            for (int j = 0; j < M; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
        }
    };
    const bool bias = p.db && k0 == 0 && k_off == 0;                        // this wave also sums dZ over the rows
    auto flush = [&](int g) {
        const int b0 = p.rows.tile_base[g], b1 = p.rows.tile_base[g + 1];
        const bool whole = b0 >= t0 && b1 <= t1;
        const int64_t slot = 2 * (int64_t)c + (b0 >= t0 ? 1 : 0);
#pragma unroll
        for (int i = 0; i < M; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int n = n0 + n_off + 32 * i + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
                if (n >= N) continue;
#pragma unroll
                for (int j = 0; j < M; ++j) {
                    const int k = k0 + k_off + 32 * j + (lane & 31);
                    if (k >= K) continue;
                    if (whole) ((T*)p.dw)[((int64_t)g * N + n) * K + k] = (T)acc[i][j][r];
                    else p.part_w[(slot * N + n) * K + k] = acc[i][j][r];
                }
                if (bias && (lane & 31) == 0) {
                    if (whole) ((T*)p.db)[(int64_t)g * N + n] = (T)accb[i][r];
                    else p.part_b[slot * N + n] = accb[i][r];
                }
            }
    };
    typename El<T>::frag ones;
#pragma unroll
    for (int e = 0; e < E; ++e) ones[e] = (T)1.0f;

    clear();
    find(0);
    load();
    find(1);
    put(0);
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
        if (s + 1 < steps) {
            load();
            find(s + 2);
        }
        const char* X = lds + (s & 1) * STAGE;
        const char* D = X + tr_bytes<T>();
#pragma unroll
        for (int u = 0; u < ROW_PIECES / 2; ++u) {
            typename El<T>::frag fx[M], fd[M];
#pragma unroll
            for (int i = 0; i < M; ++i) {
                fx[i] = tr_frag<T>(X, k_off + 32 * i, u, lane);
                fd[i] = tr_frag<T>(D, n_off + 32 * i, u, lane);
            }
#pragma unroll
            for (int i = 0; i < M; ++i)
#pragma unroll
                for (int j = 0; j < M; ++j) acc[i][j] = El<T>::mfma(fd[i], fx[j], acc[i][j]);
            if (bias)
#pragma unroll
                for (int i = 0; i < M; ++i) accb[i] = El<T>::mfma(fd[i], ones, accb[i]);
        }
        if ((s + 1) % PER_TILE == 0) {
            const int i = s / PER_TILE;
            if (i + 1 == t1 - t0 || tile_grp[i + 1] != tile_grp[i]) {
                flush(tile_grp[i]);
                clear();
            }
        }
        if (s + 1 < steps) put((s + 1) & 1);
        __syncthreads();
    }
}

// Groups whose tiles lie in several chunks: the sum of their pieces in order; groups without rows: zeros.
template <typename T>
__global__ __launch_bounds__(THREADS) void wgrad_join_kernel(WgradArgs p) {
    const int g = blockIdx.y;
    const int b0 = p.rows.tile_base[g], b1 = p.rows.tile_base[g + 1];
    const int c0 = b0 / p.chunk, c1 = b1 > b0 ? (b1 - 1) / p.chunk : c0;
    if (b1 > b0 && c0 == c1) return;
    const int64_t NK = (int64_t)p.N * p.K;
    const int64_t first = (int64_t)blockIdx.x * (THREADS * 4) + threadIdx.x;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int64_t i = first + u * THREADS;
        const bool is_w = i < NK;
        if (!is_w && !(p.db && i < NK + p.N)) continue;
        const float* part = is_w ? p.part_w + i : p.part_b + (i - NK);
        const int64_t ld = is_w ? NK : p.N;
        float sum = 0.0f;
        if (b1 > b0) {
            sum = part[(2 * (int64_t)c0 + 1) * ld];
#pragma unroll 8
            for (int c = c0 + 1; c <= c1; ++c) sum += part[2 * (int64_t)c * ld];
        }
        if (is_w) ((T*)p.dw)[g * NK + i] = (T)sum;
        else ((T*)p.db)[(int64_t)g * p.N + (i - NK)] = (T)sum;
    }
}

static inline bool sizes_ok(int64_t n, int64_t n_groups, int K, int N) {
    return n >= 0 && n <= grp::MAX_ROWS && n_groups >= 1 && n_groups <= 65535 && K >= 1 && K <= 65536 && N >= 1 && N <= 65536;
}
static inline int64_t max_tiles(int64_t n, int64_t n_groups) { return n / TILE_ROWS + n_groups + 1; }

// workgroups of a grid whose kernel spreads `work` over the eight XCDs in runs of `unit`
static inline int64_t xcd_grid(int64_t work, int64_t unit) { return ((work + unit - 1) / unit + 7) / 8 * unit * 8; }

struct WgradPlan {
    int bt, tiles_n, tiles_k, chunk;
    int64_t chunks, part_w, part_b, bytes;
};
static WgradPlan wgrad_plan(int64_t n, int64_t n_groups, int K, int N) {
    WgradPlan w = {};
    w.bt = K <= 64 && N <= 64 ? 64 : 128;
    w.tiles_n = (N + w.bt - 1) / w.bt;
    w.tiles_k = (K + w.bt - 1) / w.bt;
    const int64_t tiles = max_tiles(n, n_groups), blocks = (int64_t)w.tiles_n * w.tiles_k;
    int64_t chunks = 512 / blocks;                       // two workgroups per compute unit
    if (chunks < 1) chunks = 1;
    int64_t chunk = (tiles + chunks - 1) / chunks;
    if (chunk < 2) chunk = 2;
    if (chunk > MAX_CHUNK_TILES) chunk = MAX_CHUNK_TILES;
    w.chunk = (int)chunk;
    w.chunks = (tiles + chunk - 1) / chunk;
    // one chunk holds every group whole and leaves no pieces
    const int64_t slots = w.chunks > 1 ? 2 * w.chunks : 0;
    w.part_w = 0;
    w.part_b = (slots * N * K * 4 + 255) / 256 * 256;
    w.bytes = w.part_b + slots * N * 4;
    if (w.bytes < 256) w.bytes = 256;
    return w;
}

template <bool WT>
static int launch_linear(const LinArgs& args, int precision, bool wide, void* stream) {
    LinArgs p = args;
    const int bn = p.O <= 64 ? 64 : 128;
    p.tiles_o = (p.O + bn - 1) / bn;
    const int64_t grid = xcd_grid(max_tiles(p.rows.n, p.rows.n_groups) * p.tiles_o, 1);
    NERF_REQUIRE(grid < ((int64_t)1 << 31), NERF_E_SHAPE);
    hipStream_t st = (hipStream_t)stream;
#define NERF_LIN(T, GATE, WIDE, BN) \
    hipLaunchKernelGGL((linear_kernel<T, WT, GATE, WIDE, BN>), dim3((unsigned)grid), dim3(THREADS), 0, st, p)
#define NERF_LIN_G(T, GATE)                               \
    do {                                                  \
        if (wide && bn == 128) NERF_LIN(T, GATE, true, 128); \
        else if (wide) NERF_LIN(T, GATE, true, 64);       \
        else if (bn == 128) NERF_LIN(T, GATE, false, 128); \
        else NERF_LIN(T, GATE, false, 64);                \
    } while (0)
#define NERF_CALL(T)                                      \
    do {                                                  \
        if constexpr (WT) {                               \
            if (p.gate) NERF_LIN_G(T, true);              \
            else NERF_LIN_G(T, false);                    \
        } else {                                          \
            NERF_LIN_G(T, false);                         \
        }                                                 \
    } while (0)
    NERF_ELEM_DISPATCH(precision, NERF_CALL);
#undef NERF_CALL
#undef NERF_LIN_G
#undef NERF_LIN
    return nerf_launch_status();
}

}  // namespace gl
}  // namespace nerf

extern "C" int nerf_grouped_fwd(int64_t n, int64_t n_groups, const int32_t* order, const int32_t* offsets, const int32_t* tile_base,
                                int K, int N, const void* x, int64_t x_ld, const void* weight, const void* bias, int relu,
                                int precision, void* y, void* stream) {
    using namespace nerf;
    NERF_REQUIRE(gl::sizes_ok(n, n_groups, K, N) && x_ld >= K, NERF_E_SHAPE);
    NERF_REQUIRE(elem_ok(precision), NERF_E_DTYPE);
    if (n == 0) return NERF_OK;
    NERF_REQUIRE(offsets && tile_base && x && weight && y, NERF_E_NULL);
    const int es = elem_bytes(precision), E = 16 / es;
    NERF_REQUIRE(nerf_aligned(x, (uintptr_t)es) && nerf_aligned(weight, (uintptr_t)es) && nerf_aligned(y, (uintptr_t)es) &&
                 nerf_aligned(bias, (uintptr_t)es), NERF_E_ALIGN);
    const bool wide = K % E == 0 && N % E == 0 && x_ld % E == 0 && nerf_aligned(x, 16) && nerf_aligned(weight, 16) && nerf_aligned(y, 16);
    gl::LinArgs p = {};
    p.rows = {n, (int)n_groups, order, offsets, tile_base};
    p.C = K; p.O = N; p.a = x; p.a_ld = x_ld; p.w = weight; p.bias = bias; p.relu = relu ? 1 : 0; p.out = y;
    return gl::launch_linear<false>(p, precision, wide, stream);
}

extern "C" int nerf_grouped_bwd_data(int64_t n, int64_t n_groups, const int32_t* order, const int32_t* offsets, const int32_t* tile_base,
                                     int K, int N, const void* d_y, int64_t d_y_ld, const void* y, const void* weight, int precision,
                                     void* d_x, void* stream) {
    using namespace nerf;
    NERF_REQUIRE(gl::sizes_ok(n, n_groups, K, N) && d_y_ld >= N, NERF_E_SHAPE);
    NERF_REQUIRE(elem_ok(precision), NERF_E_DTYPE);
    if (n == 0) return NERF_OK;
    NERF_REQUIRE(offsets && tile_base && d_y && weight && d_x, NERF_E_NULL);
    const int es = elem_bytes(precision), E = 16 / es;
    NERF_REQUIRE(nerf_aligned(d_y, (uintptr_t)es) && nerf_aligned(weight, (uintptr_t)es) && nerf_aligned(d_x, (uintptr_t)es) &&
                 nerf_aligned(y, (uintptr_t)es), NERF_E_ALIGN);
    const bool wide = K % E == 0 && N % E == 0 && d_y_ld % E == 0 && nerf_aligned(d_y, 16) && nerf_aligned(weight, 16) &&
                      nerf_aligned(d_x, 16) && nerf_aligned(y, 16);
    gl::LinArgs p = {};
    p.rows = {n, (int)n_groups, order, offsets, tile_base};
    p.C = N; p.O = K; p.a = d_y; p.a_ld = d_y_ld; p.gate = y; p.w = weight; p.out = d_x;
    return gl::launch_linear<true>(p, precision, wide, stream);
}

extern "C" int64_t nerf_grouped_bwd_weights_workspace_bytes(int64_t n, int64_t n_groups, int K, int N) {
    if (!nerf::gl::sizes_ok(n, n_groups, K, N)) return NERF_E_SHAPE;
    return nerf::gl::wgrad_plan(n, n_groups, K, N).bytes;
}

extern "C" int nerf_grouped_bwd_weights(int64_t n, int64_t n_groups, const int32_t* order, const int32_t* offsets,
                                        const int32_t* tile_base, int K, int N, const void* d_y, int64_t d_y_ld, const void* y,
                                        const void* x, int64_t x_ld, int precision, void* d_weight, void* d_bias, void* workspace,
                                        int64_t workspace_bytes, void* stream) {
    using namespace nerf;
    NERF_REQUIRE(gl::sizes_ok(n, n_groups, K, N) && d_y_ld >= N && x_ld >= K, NERF_E_SHAPE);
    NERF_REQUIRE(elem_ok(precision), NERF_E_DTYPE);
    if (n == 0) return NERF_OK;
    NERF_REQUIRE(offsets && tile_base && d_y && x && d_weight && workspace, NERF_E_NULL);
    const int es = elem_bytes(precision), E = 16 / es;
    NERF_REQUIRE(nerf_aligned(d_y, (uintptr_t)es) && nerf_aligned(x, (uintptr_t)es) && nerf_aligned(y, (uintptr_t)es) &&
                 nerf_aligned(d_weight, (uintptr_t)es) && nerf_aligned(d_bias, (uintptr_t)es) && nerf_aligned(workspace, 256), NERF_E_ALIGN);
    const gl::WgradPlan w = gl::wgrad_plan(n, n_groups, K, N);
    NERF_REQUIRE(workspace_bytes >= w.bytes, NERF_E_WORKSPACE);
    const bool wide = K % E == 0 && N % E == 0 && d_y_ld % E == 0 && x_ld % E == 0 && nerf_aligned(d_y, 16) && nerf_aligned(x, 16) &&
                      nerf_aligned(y, 16);
    gl::WgradArgs p = {};
    p.rows = {n, (int)n_groups, order, offsets, tile_base};
    p.K = K; p.N = N; p.tiles_k = w.tiles_k; p.tiles_n = w.tiles_n; p.chunk = w.chunk;
    p.x_ld = x_ld; p.dy_ld = d_y_ld; p.x = x; p.dy = d_y; p.y = y; p.dw = d_weight; p.db = d_bias;
    p.part_w = (float*)((char*)workspace + w.part_w);
    p.part_b = (float*)((char*)workspace + w.part_b);
    const int64_t blocks = (int64_t)w.tiles_n * w.tiles_k;
    const int64_t grid = gl::xcd_grid(w.chunks * blocks, blocks);
    NERF_REQUIRE(grid < ((int64_t)1 << 31), NERF_E_SHAPE);
    hipStream_t st = (hipStream_t)stream;
    const dim3 join((unsigned)(((int64_t)N * K + N + gl::THREADS * 4 - 1) / (gl::THREADS * 4)), (unsigned)n_groups);
#define NERF_WG(T, GATE, WIDE, BT) \
    hipLaunchKernelGGL((gl::wgrad_kernel<T, GATE, WIDE, BT>), dim3((unsigned)grid), dim3(gl::THREADS), 0, st, p)
#define NERF_WG_G(T, GATE)                                  \
    do {                                                    \
        if (wide && w.bt == 128) NERF_WG(T, GATE, true, 128); \
        else if (wide) NERF_WG(T, GATE, true, 64);          \
        else if (w.bt == 128) NERF_WG(T, GATE, false, 128); \
        else NERF_WG(T, GATE, false, 64);                   \
    } while (0)
#define NERF_CALL(T)                                                                                   \
    do {                                                                                               \
        if (p.y) NERF_WG_G(T, true);                                                                   \
        else NERF_WG_G(T, false);                                                                      \
        hipLaunchKernelGGL(gl::wgrad_join_kernel<T>, join, dim3(gl::THREADS), 0, st, p);               \
    } while (0)
    NERF_ELEM_DISPATCH(precision, NERF_CALL);
#undef NERF_CALL
#undef NERF_WG_G
#undef NERF_WG
    return nerf_launch_status();
}
