// Rows of a table by id, scaled, and the table's gradient: per-image codes and feature tables beside the positional
// encoding.  (The reference feeds its networks encoded positions only, models/nerf.py:68-76.)
//
//   out[i] = scale * table[ids[i]]          an id outside [0, rows) gives a row of zeros
//   d_table[v] = scale * sum of d_out[i] over the i with ids[i] = v
//
// Forward: bound by memory, one 16-byte piece of a row per lane, four rows in flight per lane group.  The last piece of a row
// ends where the row does and repeats some of its columns, which are then written twice, with the same values.
// (524 288 rows of 67 bf16: forward 25 us, element by element 49; gradient 73 and 96.)
//
// Gradient: the positions come sorted by id (nerf_group_rows).  A lane group of LPR lanes sums R consecutive sorted
// positions, a lane holding VEC columns in fp32; a run of equal ids that begins and ends inside is finished at once.
// The ragged ends of a workgroup's lane groups meet in LDS, those of the workgroups in the workspace, where a second
// kernel adds them up in order of position and writes zeros for the rows that nothing reads.  No atomics: the result
// does not depend on timing, and an id that holds all positions is spread over all workgroups like any other.
// A term of the sum passes few fp32 additions however many there are: at most 64 in its lane group, G in LDS (G = 256 / LPR),
// n / (64 G^2) or 1024 / G and then G more over the workgroups.  524 288 terms of one row, fp32: 115 to 211 additions at most, error 7e-8 of the
// sum of magnitudes.
#include "elems.hpp"
#include "groups.hpp"

namespace nerf {
namespace emb {

constexpr int THREADS = 256;
constexpr int FWD_ROWS = 4;      // rows a lane group has in flight
constexpr int SMALL_N = 4096;    // positions of a call that one kernel serves
constexpr int LONG_RUN = 16;     // workgroup partials of one row above which a whole workgroup adds them up

// LPR lanes share a row; columns beyond LPR * VEC are walked by the same lanes
template <typename T, int VEC, typename ID>
__global__ __launch_bounds__(THREADS) void fwd_kernel(int64_t n, const ID* __restrict__ ids, int64_t rows, int dim, int lpr,
                                                      const T* __restrict__ table, int64_t ld, float scale, T* __restrict__ out) {
    const int groups = THREADS / lpr;
    const int sub = (int)threadIdx.x / lpr, l = (int)threadIdx.x % lpr;
    const int64_t step = (int64_t)gridDim.x * groups * FWD_ROWS;
    for (int64_t i0 = ((int64_t)blockIdx.x * groups + sub) * FWD_ROWS; i0 < n; i0 += step) {
        int64_t id[FWD_ROWS];
#pragma unroll
        for (int j = 0; j < FWD_ROWS; ++j) id[j] = i0 + j < n ? (int64_t)ids[i0 + j] : -1;
        for (int c0 = l * VEC; c0 < dim; c0 += lpr * VEC) {
            const int c = min(c0, dim - VEC);
            Pack<T, VEC> x[FWD_ROWS];
#pragma unroll
            for (int j = 0; j < FWD_ROWS; ++j) {
                const bool ok = id[j] >= 0 && id[j] < rows;
                if (ok) x[j] = load_any<T, VEC>(table + id[j] * ld + c);
                else
#pragma unroll
                    for (int v = 0; v < VEC; ++v) x[j].v[v] = (T)0.0f;
            }
#pragma unroll
            for (int j = 0; j < FWD_ROWS; ++j) {
                if (i0 + j >= n) break;
                const bool ok = id[j] >= 0 && id[j] < rows;
                Pack<T, VEC> y;
#pragma unroll
                for (int v = 0; v < VEC; ++v) y.v[v] = ok ? (T)((float)x[j].v[v] * scale) : (T)0.0f;
                store_any<T, VEC>(out + (i0 + j) * dim + c, y);
            }
        }
    }
}

struct BwdArgs {
    int64_t n, rows;
    int dim, lpr, per;             // per: sorted positions of one lane group
    const int32_t *order, *offsets, *keys;
    float scale;
    float* part;                   // [2 * workgroups][dim]: slot 2w a run that came in from the left of workgroup w,
};                                 // slot 2w + 1 one that began in it and goes on to the right

template <typename T, int VEC>
__device__ __forceinline__ void write_row(T* d_table, int64_t row, int dim, int col, const float (&acc)[VEC], float scale) {
    Pack<T, VEC> y;
#pragma unroll
    for (int v = 0; v < VEC; ++v) y.v[v] = (T)(acc[v] * scale);
    store_any<T, VEC>(d_table + row * dim + col, y);
}

template <int VEC>
__device__ __forceinline__ void write_part(float* part, int64_t slot, int dim, int col, const float (&acc)[VEC]) {
    Pack<float, VEC> y;
#pragma unroll
    for (int v = 0; v < VEC; ++v) y.v[v] = acc[v];
    if constexpr (VEC == 8) {
        Pack<float, 4> a, b;
#pragma unroll
        for (int v = 0; v < 4; ++v) { a.v[v] = acc[v]; b.v[v] = acc[4 + v]; }
        store_any<float, 4>(part + slot * dim + col, a);
        store_any<float, 4>(part + slot * dim + col + 4, b);
    } else {
        store_any<float, VEC>(part + slot * dim + col, y);
    }
}

template <int VEC>
__device__ __forceinline__ void add_part(float (&acc)[VEC], const float* p) {
    if constexpr (VEC == 8) {
        const Pack<float, 4> a = load_any<float, 4>(p), b = load_any<float, 4>(p + 4);
#pragma unroll
        for (int v = 0; v < 4; ++v) { acc[v] += a.v[v]; acc[4 + v] += b.v[v]; }
    } else {
        const Pack<float, VEC> a = load_any<float, VEC>(p);
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[v] += a.v[v];
    }
}

// Four workgroups to a compute unit: 16-bit tensors spill one register for it, and are no slower (524 288 x 128 fp16, the whole
// gradient: 101 us, 103 with three and no spill).
template <typename T, int VEC>
__global__ __launch_bounds__(THREADS, 4) void bwd_sum_kernel(BwdArgs a, const T* __restrict__ d_out, int64_t ld, T* __restrict__ d_table) {
    constexpr int BATCH = 8;
    __shared__ float head[THREADS * VEC], tail[THREADS * VEC];
    __shared__ int head_state[THREADS], tail_key[THREADS];         // head: 0 none, 1 ends in its lane group, 2 goes on
    const int lpr = a.lpr, groups = THREADS / lpr;
    const int sub = (int)threadIdx.x / lpr, l = (int)threadIdx.x % lpr;
    const int col0 = ((int)blockIdx.y * lpr + l) * VEC, col = min(col0, a.dim - VEC);
    const bool on = col0 < a.dim;
    const int64_t nv = a.offsets[a.rows];                          // positions behind it belong to no row
    const int64_t p0 = ((int64_t)blockIdx.x * groups + sub) * a.per;
    const int64_t p1 = p0 + a.per < nv ? p0 + a.per : nv;
    int hstate = 0, tkey = -1;
    if (p0 < p1) {
        float acc[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[v] = 0.0f;
        int key = a.keys[p0];
        bool from_left = p0 > 0 && a.keys[p0 - 1] == key;
        // rows of d_out are requested a batch ahead, their numbers two
        int k[BATCH], next_k[BATCH], row[BATCH];
        Pack<T, VEC> x[BATCH], next_x[BATCH];
        auto numbers = [&](int64_t p) {
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                const int64_t q = p + j < p1 ? p + j : p1 - 1;
                next_k[j] = a.keys[q];
                row[j] = a.order[q];
            }
        };
        auto request = [&]() {
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                k[j] = next_k[j];
                if (on) next_x[j] = load_any<T, VEC>(d_out + row[j] * ld + col);
            }
        };
        numbers(p0);
        request();
        numbers(p0 + BATCH);
        for (int64_t p = p0; p < p1; p += BATCH) {
            int now[BATCH];
#pragma unroll
            for (int j = 0; j < BATCH; ++j) { now[j] = k[j]; x[j] = next_x[j]; }
            request();
            numbers(p + 2 * BATCH);
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                if (p + j >= p1) break;
                if (now[j] != key) {                               // the run of `key` ends here
                    if (from_left) {
                        hstate = 1;
                        if (on)
#pragma unroll
                            for (int v = 0; v < VEC; ++v) head[threadIdx.x * VEC + v] = acc[v];
                    } else if (on) {
                        write_row<T, VEC>(d_table, key, a.dim, col, acc, a.scale);
                    }
                    from_left = false;
                    key = now[j];
#pragma unroll
                    for (int v = 0; v < VEC; ++v) acc[v] = 0.0f;
                }
                if (on)
#pragma unroll
                    for (int v = 0; v < VEC; ++v) acc[v] += (float)x[j].v[v];
            }
        }
        const bool goes_on = p1 < nv && a.keys[p1] == key;
        if (from_left) {
            hstate = goes_on ? 2 : 1;
            if (on)
#pragma unroll
                for (int v = 0; v < VEC; ++v) head[threadIdx.x * VEC + v] = acc[v];
        } else if (goes_on) {
            tkey = key;
            if (on)
#pragma unroll
                for (int v = 0; v < VEC; ++v) tail[threadIdx.x * VEC + v] = acc[v];
        } else if (on) {
            write_row<T, VEC>(d_table, key, a.dim, col, acc, a.scale);
        }
    }
    if (l == 0) { head_state[sub] = hstate; tail_key[sub] = tkey; }
    __syncthreads();
    if (sub != 0 || !on) return;
    float acc[VEC];
    bool open = false, from_left = false;
    int key = -1;
    for (int g = 0; g < groups; ++g) {
        const int at = (g * lpr + l) * VEC;
        const int hs = head_state[g], tk = tail_key[g];
        if (hs) {
            if (!open) {                                           // g == 0: the run comes from an earlier workgroup
                from_left = open = true;
#pragma unroll
                for (int v = 0; v < VEC; ++v) acc[v] = 0.0f;
            }
#pragma unroll
            for (int v = 0; v < VEC; ++v) acc[v] += head[at + v];
            if (hs == 1) {
                if (from_left) write_part<VEC>(a.part, 2 * (int64_t)blockIdx.x, a.dim, col, acc);
                else write_row<T, VEC>(d_table, key, a.dim, col, acc, a.scale);
                open = false;
            }
        }
        if (tk >= 0) {
            open = true;
            from_left = false;
            key = tk;
#pragma unroll
            for (int v = 0; v < VEC; ++v) acc[v] = tail[at + v];
        }
    }
    if (open) write_part<VEC>(a.part, 2 * (int64_t)blockIdx.x + (from_left ? 0 : 1), a.dim, col, acc);
}

// Rows whose positions span several workgroups of bwd_sum_kernel, and rows that hold none.
template <typename T, int VEC>
__global__ __launch_bounds__(THREADS) void bwd_join_kernel(BwdArgs a, T* __restrict__ d_table) {
    __shared__ float red[THREADS * VEC];
    const int lpr = a.lpr, groups = THREADS / lpr;
    const int sub = (int)threadIdx.x / lpr, l = (int)threadIdx.x % lpr;
    const int col0 = ((int)blockIdx.y * lpr + l) * VEC, col = min(col0, a.dim - VEC);
    const bool on = col0 < a.dim;
    const int64_t span = (int64_t)groups * a.per;
    const int64_t row0 = (int64_t)blockIdx.x * groups;
    const int64_t row = row0 + sub;
    bool any_long = false;
    if (row < a.rows) {
        const int64_t s = a.offsets[row], e = a.offsets[row + 1];
        float acc[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[v] = 0.0f;
        if (s == e) {
            if (on) {
                Pack<T, VEC> zero;
#pragma unroll
                for (int v = 0; v < VEC; ++v) zero.v[v] = (T)0.0f;
                store_any<T, VEC>(d_table + row * a.dim + col, zero);
            }
        } else {
            const int64_t w0 = s / span, w1 = (e - 1) / span;
            any_long = w1 - w0 >= LONG_RUN;
            if (w1 > w0 && !any_long && on) {
                add_part<VEC>(acc, a.part + (2 * w0 + 1) * a.dim + col);
                for (int64_t w = w0 + 1; w <= w1; ++w) add_part<VEC>(acc, a.part + 2 * w * a.dim + col);
                write_row<T, VEC>(d_table, row, a.dim, col, acc, a.scale);
            }
        }
    }
    if (!__syncthreads_or(any_long)) return;
    for (int g = 0; g < groups; ++g) {
        if (row0 + g >= a.rows) break;
        const int64_t s = a.offsets[row0 + g], e = a.offsets[row0 + g + 1];
        if (s == e) continue;
        const int64_t w0 = s / span, w1 = (e - 1) / span;
        if (w1 - w0 < LONG_RUN) continue;
        float acc[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[v] = 0.0f;
        if (on) {
            // lane group `sub` takes a run of consecutive workgroups, so the order of the sum is that of the positions
            const int64_t cnt = (w1 - w0 + 1 + groups - 1) / groups;
            const int64_t from = w0 + sub * cnt, to = from + cnt < w1 + 1 ? from + cnt : w1 + 1;
#pragma unroll 8
            for (int64_t w = from; w < to; ++w) add_part<VEC>(acc, a.part + (2 * w + (w == w0 ? 1 : 0)) * a.dim + col);
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) red[threadIdx.x * VEC + v] = acc[v];
        __syncthreads();
        if (sub == 0 && on) {
            for (int k = 1; k < groups; ++k)
#pragma unroll
                for (int v = 0; v < VEC; ++v) acc[v] += red[(k * lpr + l) * VEC + v];
            write_row<T, VEC>(d_table, row0 + g, a.dim, col, acc, a.scale);
        }
        __syncthreads();
    }
}

// Few positions and few rows: a workgroup per table row looks through all ids, keeps the positions that name its row (in
// order, each wave its own quarter) and sums their rows of d_out, one launch instead of five.  1024 positions over 100 rows
// of 48 fp32: 5 us, grouped first 16; small_call() says where it stops paying.
template <typename T, int VEC, typename ID>
__global__ __launch_bounds__(THREADS) void bwd_small_kernel(int n, const ID* __restrict__ ids, int dim, int lpr, const T* __restrict__ d_out,
                                                            int64_t ld, float scale, T* __restrict__ d_table) {
    constexpr int ROUNDS = SMALL_N / THREADS;
    __shared__ int list[SMALL_N];
    __shared__ int count[THREADS / 64];
    __shared__ float red[THREADS * VEC];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row = blockIdx.x, quarter = (n + THREADS - 1) / THREADS * 64;
    ID id[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int p = wave * quarter + r * 64 + lane;
        id[r] = r * 64 < quarter && p < n ? ids[p] : (ID)-1;
    }
    int cnt = 0;
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const bool mine = id[r] == (ID)row;
        const unsigned long long m = __ballot(mine);
        if (mine) list[wave * quarter + cnt + __popcll(m & ((1ull << lane) - 1ull))] = wave * quarter + r * 64 + lane;
        cnt += __popcll(m);
    }
    if (lane == 0) count[wave] = cnt;
    const bool any = __syncthreads_or(cnt);                        // a row that nothing reads gets zeros, whatever the scale is
    __syncthreads();
    const int groups = THREADS / lpr, sub = (int)threadIdx.x / lpr, l = (int)threadIdx.x % lpr;
    for (int col0 = l * VEC; col0 - l * VEC < dim; col0 += lpr * VEC) {
        const bool on = col0 < dim;
        const int col = min(col0, dim - VEC);
        float acc[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) acc[v] = 0.0f;
        int at = sub;                                              // positions sub, sub + groups, .. of the four lists in a row
        for (int w = 0; w < THREADS / 64; ++w) {
            for (; at < count[w]; at += groups) {
                if (!on) continue;
                const Pack<T, VEC> x = load_any<T, VEC>(d_out + list[w * quarter + at] * ld + col);
#pragma unroll
                for (int v = 0; v < VEC; ++v) acc[v] += (float)x.v[v];
            }
            at -= count[w];
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) red[threadIdx.x * VEC + v] = acc[v];
        __syncthreads();
        if (sub == 0 && on) {
            for (int k = 1; k < groups; ++k)
#pragma unroll
                for (int v = 0; v < VEC; ++v) acc[v] += red[(k * lpr + l) * VEC + v];
            write_row<T, VEC>(d_table, row, dim, col, acc, any ? scale : 0.0f);
        }
        __syncthreads();
    }
}

// up to four million comparisons of ids with rows, at most 4096 of each: 4096 positions over 256 rows take 5 us, over 1024 rows 7
// (grouped first 24 to 27), 64 positions over 4096 rows 10 (18)
static inline bool small_call(int64_t n, int64_t rows) { return n <= SMALL_N && rows <= SMALL_N && n * rows <= ((int64_t)1 << 22); }

static inline int lanes_per_row(int64_t dim, int vec) {
    int l = 4;
    while (l < 64 && (int64_t)l * vec < dim) l <<= 1;
    return l;
}

// sorted positions of a lane group: enough workgroups to fill the chip (1024), few enough partial sums
static inline int positions_per_group(int64_t n, int groups) {
    int64_t per = (n / ((int64_t)groups * 1024) + 7) / 8 * 8;
    if (per < 8) per = 8;
    if (per > 64) per = 64;
    return (int)per;
}

static inline bool sizes_ok(int64_t n, int64_t rows, int64_t dim) {
    return n >= 0 && n <= grp::MAX_ROWS && rows >= 1 && rows <= grp::MAX_GROUPS && dim >= 1 && dim <= (1 << 20);
}

}  // namespace emb
}  // namespace nerf

extern "C" int nerf_embed_fwd(int64_t n, const void* ids, int id_bytes, int64_t rows, int64_t dim, const void* table, int64_t table_ld,
                              float scale, int precision, void* out, void* stream) {
    using namespace nerf;
    NERF_REQUIRE(emb::sizes_ok(n, rows, dim) && table_ld >= dim, NERF_E_SHAPE);
    NERF_REQUIRE(elem_ok(precision) && (id_bytes == 4 || id_bytes == 8), NERF_E_DTYPE);
    if (n == 0) return NERF_OK;
    NERF_REQUIRE(ids && table && out, NERF_E_NULL);
    const int es = elem_bytes(precision), full = 16 / es;
    NERF_REQUIRE(nerf_aligned(ids, (uintptr_t)id_bytes) && nerf_aligned(table, (uintptr_t)es) && nerf_aligned(out, (uintptr_t)es), NERF_E_ALIGN);
    const bool wide = dim >= full;
    const int lpr = emb::lanes_per_row(dim, wide ? full : 1);
    const int64_t per_block = (int64_t)(emb::THREADS / lpr) * emb::FWD_ROWS;
    int64_t blocks = (n + per_block - 1) / per_block;
    if (blocks > 16384) blocks = 16384;
    hipStream_t st = (hipStream_t)stream;
#define NERF_FWD(T, V, ID)                                                                                                      \
    hipLaunchKernelGGL((emb::fwd_kernel<T, V, ID>), dim3((unsigned)blocks), dim3(emb::THREADS), 0, st, n, (const ID*)ids, rows, (int)dim, \
                       lpr, (const T*)table, table_ld, scale, (T*)out)
#define NERF_CALL(T)                                                                      \
    do {                                                                                  \
        if (wide && id_bytes == 8) NERF_FWD(T, full_vec<T>(), int64_t);                   \
        else if (wide) NERF_FWD(T, full_vec<T>(), int32_t);                               \
        else if (id_bytes == 8) NERF_FWD(T, 1, int64_t);                                  \
        else NERF_FWD(T, 1, int32_t);                                                     \
    } while (0)
    NERF_ELEM_DISPATCH(precision, NERF_CALL);
#undef NERF_CALL
#undef NERF_FWD
    return nerf_launch_status();
}

namespace nerf {
namespace emb {

struct BwdPlan { int64_t order, offsets, keys, part, group, bytes; };     // byte offsets in the workspace
static BwdPlan bwd_plan(int64_t n, int64_t rows, int64_t dim) {
    BwdPlan p = {};
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    int64_t part = 0;                       // over the access widths, which the pointers decide
    for (int vec : {1, 4, 8}) {
        const int groups = THREADS / lanes_per_row(dim, vec);
        const int64_t span = (int64_t)groups * positions_per_group(n, groups);
        const int64_t b = 2 * ((n + span - 1) / span) * dim * 4;
        if (b > part) part = b;
    }
    p.order = take(4 * n);
    p.offsets = take(4 * (rows + 1));
    p.keys = take(4 * n);
    p.part = take(part);
    p.group = take(grp::workspace_bytes(n, rows));
    p.bytes = at;
    return p;
}

}  // namespace emb
}  // namespace nerf

extern "C" int64_t nerf_embed_bwd_workspace_bytes(int64_t n, int64_t rows, int64_t dim) {
    if (!nerf::emb::sizes_ok(n, rows, dim)) return NERF_E_SHAPE;
    return nerf::emb::small_call(n, rows) ? 0 : nerf::emb::bwd_plan(n, rows, dim).bytes;
}

extern "C" int nerf_embed_bwd(int64_t n, const void* ids, int id_bytes, int64_t rows, int64_t dim, const void* d_out, int64_t d_out_ld,
                              float scale, int precision, void* d_table, void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace nerf;
    NERF_REQUIRE(emb::sizes_ok(n, rows, dim) && d_out_ld >= dim, NERF_E_SHAPE);
    NERF_REQUIRE(elem_ok(precision) && (id_bytes == 4 || id_bytes == 8), NERF_E_DTYPE);
    if (n == 0) return NERF_OK;
    const bool small = emb::small_call(n, rows);
    NERF_REQUIRE(ids && d_out && d_table && (workspace || small), NERF_E_NULL);
    const int es = elem_bytes(precision), full = 16 / es;
    NERF_REQUIRE(nerf_aligned(ids, (uintptr_t)id_bytes) && nerf_aligned(d_out, (uintptr_t)es) && nerf_aligned(d_table, (uintptr_t)es) &&
                 nerf_aligned(workspace, 256), NERF_E_ALIGN);
    const emb::BwdPlan plan = emb::bwd_plan(n, rows, dim);
    NERF_REQUIRE(small || workspace_bytes >= plan.bytes, NERF_E_WORKSPACE);
    char* ws = (char*)workspace;
    hipStream_t st = (hipStream_t)stream;
    int32_t *order = (int32_t*)(ws + plan.order), *offsets = (int32_t*)(ws + plan.offsets), *keys = (int32_t*)(ws + plan.keys);
    const bool wide = dim >= full;
    const int vec = wide ? full : 1, lpr = emb::lanes_per_row(dim, vec);
    if (small) {
#define NERF_SMALL(T, V, ID)                                                                                                      \
    hipLaunchKernelGGL((emb::bwd_small_kernel<T, V, ID>), dim3((unsigned)rows), dim3(emb::THREADS), 0, st, (int)n, (const ID*)ids, (int)dim, \
                       lpr, (const T*)d_out, d_out_ld, scale, (T*)d_table)
#define NERF_CALL(T)                                                                      \
    do {                                                                                  \
        if (wide && id_bytes == 8) NERF_SMALL(T, full_vec<T>(), int64_t);                 \
        else if (wide) NERF_SMALL(T, full_vec<T>(), int32_t);                             \
        else if (id_bytes == 8) NERF_SMALL(T, 1, int64_t);                                \
        else NERF_SMALL(T, 1, int32_t);                                                   \
    } while (0)
        NERF_ELEM_DISPATCH(precision, NERF_CALL);
#undef NERF_CALL
#undef NERF_SMALL
        return nerf_launch_status();
    }
    const int rc = grp::launch_group_rows(n, ids, id_bytes, rows, order, offsets, nullptr, keys, ws + plan.group, st);
    if (rc != NERF_OK) return rc;
    emb::BwdArgs a = {};
    a.n = n; a.rows = rows; a.dim = (int)dim;
    a.lpr = lpr;
    const int groups = emb::THREADS / a.lpr;
    a.per = emb::positions_per_group(n, groups);
    a.order = order; a.offsets = offsets; a.keys = keys; a.scale = scale; a.part = (float*)(ws + plan.part);
    const int64_t span = (int64_t)groups * a.per;
    const unsigned cols = (unsigned)((dim + (int64_t)a.lpr * vec - 1) / ((int64_t)a.lpr * vec));
    const dim3 g1((unsigned)((n + span - 1) / span), cols), g2((unsigned)((rows + groups - 1) / groups), cols), block(emb::THREADS);
#define NERF_BWD(T, V)                                                                                                        \
    do {                                                                                                                      \
        hipLaunchKernelGGL((emb::bwd_sum_kernel<T, V>), g1, block, 0, st, a, (const T*)d_out, d_out_ld, (T*)d_table);          \
        hipLaunchKernelGGL((emb::bwd_join_kernel<T, V>), g2, block, 0, st, a, (T*)d_table);                                    \
    } while (0)
#define NERF_CALL(T)                            \
    do {                                        \
        if (wide) NERF_BWD(T, full_vec<T>());   \
        else NERF_BWD(T, 1);                    \
    } while (0)
    NERF_ELEM_DISPATCH(precision, NERF_CALL);
#undef NERF_CALL
#undef NERF_BWD
    return nerf_launch_status();
}
