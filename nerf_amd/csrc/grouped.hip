// Linear layers of many sub-networks over rows grouped by id: row i belongs to group g(i) and
//   y_i = act(W_g x_i + b_g),   dX_i = W_g^T dZ_i,   dW_g = sum_i dZ_i x_i^T,   db_g = sum_i dZ_i,   dZ = dY [y > 0].
// The reference has one network for all points (models/nerf.py:155-209); here the points of one call are dealt out to
// sub-networks (a spatial grid, a router), each with as many points as fall to it.
//
// Rows stay where they are: a tile is 128 consecutive positions of the grouped order, and the kernels read and write
// row order[position] of the ordinary tensors (a row is one or more whole cache lines, so gathering costs nothing).  The
// number of tiles is known on the device only: the grid is the upper bound n / 128 + groups + 1 and a workgroup finds its
// group in tile_base, the running number of tiles, with a 64-wide comparison.
//
// Operands in whole aligned 16-byte pieces are copied into a ring of LDS buffers by the memory system itself
// (global_load_lds, 16 bytes per lane) and multiplied by persistent workgroups, one per compute unit (stream_kernel,
// wgrad_stream_kernel): v_mfma_f32_32x32x16_{bf16,f16} or, in fp32, v_mfma_f32_32x32x2_f32 (exact products, fp32 sums).
// Anything else goes through registers, one workgroup per tile (linear_kernel, wgrad_kernel), or is copied to whole pieces
// first (pad_plan).
//
// Bounds: 256 -> 256 features move 1 KiB per row for 128 kflop, memory at 16 bits (196 608 rows, inputs from memory: forward
// 70 us, data gradient 66, weight gradient 67, over a floor of 39, 39 and 28; inputs partly in the last-level cache 56, 54 and 57)
// and the fp32 matrix instructions at 32 (65 536 rows: 91, 93 and 103 us over 56, matrix pipes 55 % busy).  1024 -> 1024 features
// are bound by the copies into LDS, 33 to 37 bytes per ns and compute unit (65 536 rows fp16: forward 165 to 180 us with one group,
// 0.76 to 0.83 PFLOP/s where a large library product reaches 1.06; 190 to 204 with 64 uneven ones; matrix pipes 38 % busy).
//
// A 16-byte piece holds the values of consecutive contraction indices of one row; operands whose contraction index is the
// row (W in dX, both in dW) are read with ds_read_b64_tr_b16, which hands a lane four rows of its column, or in fp32 with
// four 4-byte reads.  Pieces are permuted within a row (by the address they are copied from) so that the lanes of one LDS
// cycle fall on different banks.
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
// Workgroups in one direction of a grid: the runtime cuts off what passes 2^32 threads, without an error.  A multiple of the
// eight XCDs that leaves room for workgroups of up to 512 threads.
constexpr int64_t MAX_GRID = (int64_t)1 << 22;

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

// ---- row-major tile, contraction index = row: [step_len rows][COLS columns] -----------------------------------
// 16-bit: a transposing read takes 64 bytes of four rows, which go to different 64-byte windows; fp32: lanes 0-31 read a
// row and lanes 32-63 the fourth one after it, which go to different halves of the banks
template <typename T, int COLS>
__device__ __forceinline__ int tr_swap(int row) {
    if constexpr (sizeof(T) == 2) return (row & (COLS < 128 ? 1 : 3)) << 2;
    else return ((row >> 2) & 1) << 3;
}
template <typename T, int COLS>
__device__ __forceinline__ int tr_addr(int row, int q) { return row * (COLS * (int)sizeof(T)) + ((q ^ tr_swap<T, COLS>(row)) << 4); }
template <typename T, int COLS> constexpr int tr_bytes() { return step_len<T>() * COLS * (int)sizeof(T); }

// where a lane begins to read its fragment of columns col0 .. col0 + 31 in product step s
template <typename T, int COLS>
__device__ __forceinline__ int tr_lane(int col0, int s, int lane) {
    if constexpr (sizeof(T) == 2) {
        const int row = 16 * s + 8 * (lane >> 5) + ((lane & 15) >> 2), col = col0 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
        return tr_addr<T, COLS>(row, col >> 3) + ((col >> 2) & 1) * 8;
    } else {
        const int col = col0 + (lane & 31);
        return tr_addr<T, COLS>(8 * s + 4 * (lane >> 5), col >> 2) + (col & 3) * 4;
    }
}

template <typename T, int COLS>
__device__ __forceinline__ typename El<T>::frag tr_frag(const char* tile, int col0, int s, int lane) {
    const char* at = tile + tr_lane<T, COLS>(col0, s, lane);
    if constexpr (sizeof(T) == 2) {
        typedef __attribute__((address_space(3))) s16x4* lds_ptr;
        struct Two { s16x4 lo, hi; } f;
        f.lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)at);
        f.hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(at + 4 * COLS * (int)sizeof(T)));    // rows 4 apart share their permutation
        return __builtin_bit_cast(typename El<T>::frag, f);
    } else {
        f32x4 f;
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = *reinterpret_cast<const float*>(at + j * COLS * 4);        // so do four rows in a run
        return f;
    }
}

// ---- copies straight into LDS: lane l of a wave fills bytes 16 l .. of the 1 KiB at `to` (wave-uniform) -------------
typedef __attribute__((address_space(1))) const char gbl_char;
typedef __attribute__((address_space(3))) char lds_char;
__device__ __constant__ const float4 ZERO_PIECE = {0.0f, 0.0f, 0.0f, 0.0f};      // read where an operand has nothing
__device__ __forceinline__ void copy_piece(const void* from, char* to) {
    __builtin_amdgcn_global_load_lds((gbl_char*)from, (lds_char*)to, 16, 0, 0);
}

// ---- pieces from memory ---------------------------------------------------------------------------------------
// columns c .. of a row that has `cols` of them; zero behind its end and when !ok.  The row may begin anywhere (memory
// instructions take any address that its elements are aligned to).  The last piece of a row is read where it ends and
// shifted into place, so nothing behind the row is touched; rows shorter than a piece go element by element.
template <typename T>
__device__ __forceinline__ Pack<T, piece<T>()> load_piece(const T* row, int c, int cols, bool ok) {
    constexpr int E = piece<T>();
    struct __attribute__((packed, aligned(sizeof(T)))) Any { unsigned long long lo, hi; };
    Pack<T, E> p;
    if (cols < E) {
#pragma unroll
        for (int e = 0; e < E; ++e) p.v[e] = ok && c + e < cols ? row[c + e] : (T)0.0f;
        return p;
    }
    const int over = c + E - cols;                                          // elements of the piece behind the row
    const Any raw = *reinterpret_cast<const Any*>(row + (over > 0 ? cols - E : c));
    unsigned long long lo = raw.lo, hi = raw.hi;
    if (over > 0) {
        const int bits = min(over, E) * (int)sizeof(T) * 8;
        if (bits >= 64) {
            lo = bits == 128 ? 0 : hi >> (bits - 64);
            hi = 0;
        } else {
            lo = (lo >> bits) | (hi << (64 - bits));
            hi >>= bits;
        }
    }
    if (!ok) lo = hi = 0;
    struct Two { unsigned long long lo, hi; } two = {lo, hi};
    return __builtin_bit_cast(Pack<T, E>, two);
}

// columns c .. of a row of `cols`, written; nothing behind the row is touched
template <typename T>
__device__ __forceinline__ void put_row_piece(T* row, int c, int cols, const Pack<T, piece<T>()>& v) {
    struct __attribute__((packed, aligned(sizeof(T)))) Any { unsigned long long lo, hi; };
    if (c + piece<T>() <= cols) *reinterpret_cast<Any*>(row + c) = __builtin_bit_cast(Any, v);
    else
#pragma unroll
        for (int e = 0; e < piece<T>(); ++e)
            if (c + e < cols) row[c + e] = v.v[e];
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

// ReLU with least = 0 and no sign bit in `bits` (keeps a NaN, without its sign); the identity with -inf and all bits
__device__ __forceinline__ float relu_or_not(float v, float least, unsigned bits) {
    return __builtin_bit_cast(float, __builtin_bit_cast(unsigned, v < least ? 0.0f : v) & bits);
}

struct Rows {
    int64_t n;
    int n_groups, most_tiles;
    const int32_t *order, *offsets, *tile_base;
};

// row of a position; -1 for an entry that is no row
__device__ __forceinline__ int row_at(const Rows& r, int64_t pos) {
    const int row = r.order[pos];
    return row >= 0 && row < r.n ? row : -1;
}

struct LinArgs {
    Rows rows;
    int C, O, tiles_o;           // contraction length, outputs, output tiles
    int grid_row;                // register form: workgroups per XCD in one row of the grid
    int64_t a_ld;
    int64_t w_ld, w_gs;          // elements between rows and between groups of w
    int w_rows;                  // rows of w where they are the contraction index (C is a whole number of pieces)
    const void *a, *w, *bias;
    int relu;
    void* out;
};

// A tile of a call: group, first position, rows, first output.  Up to 62 groups the lanes of a wave hold both tables, one
// round trip for the whole call; above, a tile costs two or three.
struct Tile {
    int64_t pos0;
    int group, count, o0;
};
struct Tables {
    int base, off, total, lane;
    __device__ __forceinline__ Tables(const Rows& r, int lane_) : base(0), off(0), lane(lane_) {
        if (r.n_groups < 63) {
            base = r.tile_base[min(lane, r.n_groups + 1)];
            off = r.offsets[min(lane, r.n_groups)];
            total = __builtin_amdgcn_readlane(base, r.n_groups + 1);
        } else {
            total = r.tile_base[r.n_groups + 1];
        }
        total = grp::checked_tiles(total, r.most_tiles);
    }
    __device__ __forceinline__ Tile tile(const Rows& r, int64_t at, int tiles_o, int bn) const {
        const int G = r.n_groups;
        Tile t;
        const int i = __builtin_amdgcn_readfirstlane((int)(at / tiles_o));
        t.o0 = (int)(at % tiles_o) * bn;
        int first, begin, end;
        if (G < 63) {
            t.group = max((int)__popcll(__ballot(lane <= G && base <= i)) - 1, 0);
            first = __builtin_amdgcn_readlane(base, t.group);
            begin = __builtin_amdgcn_readlane(off, t.group);
            end = __builtin_amdgcn_readlane(off, min(t.group + 1, G));
        } else {
            t.group = grp::group_of_tile(r.tile_base, G, i, lane);
            first = r.tile_base[t.group];
            begin = r.offsets[t.group];
            end = r.offsets[min(t.group + 1, G)];
        }
        const grp::Span span = grp::checked_span(begin + ((int64_t)i - first) * TILE_ROWS, t.group < G ? (int64_t)end : r.n, r.n);
        t.pos0 = span.pos;
        t.count = span.count;
        return t;
    }
};

// ---- streaming form: operands in whole aligned 16-byte pieces, outputs at any alignment ------------------------------------------------------
// out[row][o] = sum_c a[row][c] w_g(o, c).  WT = false: w_g is [O][C] (the layer); WT = true: w_g is [C][O] (its data
// gradient).  One workgroup of eight waves per compute unit for the whole call.  It owns a run of consecutive items (128
// rows x BN outputs) and streams their contraction steps without a gap between items: the memory system copies step s + 2
// into a ring of three LDS buffers (global_load_lds, 16 bytes per lane) while step s is multiplied; one barrier per step.
//
// vmcnt counts copies and stores in the order they were issued, so a step waits for its own copies only, with the number
// of younger copies and stores left outstanding.  For that count to be known, every wave issues the same stores for every
// item: a position behind a tile's rows repeats the tile's last row, outputs behind the last piece repeat that piece
// (out_of), and what they store is what is there already.  LDS is read by inline asm (reads and their wait in one block), because the
// compiler would wait for every copy in flight in front of a read it can see.
//
// The accumulators hold outputs down and rows across: a lane's four consecutive registers are consecutive outputs of one
// row, and one exchange between the wave's halves (v_permlane32_swap) makes them eight, a 16-byte store.
constexpr int ST_THREADS = 512;
// items whose rows and bias are in LDS at a time; 64 outputs leave room for two workgroups in a compute unit's LDS
// (65 536 rows 256 -> 256 fp32, forward in short bursts of calls: 102 us with two, 111 with one)
template <int BN> constexpr int st_items() { return BN == 64 ? 8 : 12; }

// Output number of place o.  The last piece of a row ends where the row does, so it may repeat outputs of the one before, and
// places behind it repeat it: the same values are stored again.
template <int E>
__device__ __forceinline__ int out_of(int o, int O) {
    const int first = o / E * E;
    return first + E <= O ? o : O - E + (o - first);
}

template <int N>
__device__ __forceinline__ void wait_copies() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ int lds_int(unsigned at) {
    int v;
    asm volatile("ds_read_b32 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(v) : "v"(at) : "memory");
    return v;
}
__device__ __forceinline__ f32x4 lds_quad(unsigned at) {
    f32x4 v;
    asm volatile("ds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(v) : "v"(at) : "memory");
    return v;
}

// The fragments of one product step, all requested before the one wait.  a: MI row tiles 32 rows (4 KiB) apart from one
// address; b: NJ output tiles, 4 KiB apart (NT).
template <typename F, int MI, int NJ>
__device__ __forceinline__ void read_nt(F (&a)[MI], F (&b)[NJ], unsigned pa, unsigned pb) {
    if constexpr (MI == 2 && NJ == 2)
        asm volatile("ds_read_b128 %0, %4\n\tds_read_b128 %2, %5\n\tds_read_b128 %1, %4 offset:4096\n\tds_read_b128 %3, %5 offset:4096\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(a[0]), "=&v"(a[1]), "=&v"(b[0]), "=&v"(b[1]) : "v"(pa), "v"(pb) : "memory");
    else if constexpr (MI == 2 && NJ == 1)
        asm volatile("ds_read_b128 %0, %3\n\tds_read_b128 %2, %4\n\tds_read_b128 %1, %3 offset:4096\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(a[0]), "=&v"(a[1]), "=&v"(b[0]) : "v"(pa), "v"(pb) : "memory");
    else
        asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %3\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(a[0]), "=&v"(b[0]) : "v"(pa), "v"(pb) : "memory");
}
template <typename F, int MI>
__device__ __forceinline__ void read_rows(F (&a)[MI], unsigned pa) {
    if constexpr (MI == 2)
        asm volatile("ds_read_b128 %0, %2\n\tds_read_b128 %1, %2 offset:4096\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(a[0]), "=&v"(a[1]) : "v"(pa) : "memory");
    else
        asm volatile("ds_read_b128 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(a[0]) : "v"(pa) : "memory");
}
// A transposed fragment: two reads four rows apart (16-bit) or one per row (fp32; four rows share their permutation)
template <typename T, int PITCH>
__device__ __forceinline__ typename El<T>::frag read_tr(unsigned at0) {
    if constexpr (sizeof(T) == 2) {
        struct Two { s16x4 lo, hi; } f;
        asm volatile("ds_read_b64_tr_b16 %0, %2\n\tds_read_b64_tr_b16 %1, %2 offset:%3\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(f.lo), "=&v"(f.hi) : "v"(at0), "n"(4 * PITCH) : "memory");
        return __builtin_bit_cast(typename El<T>::frag, f);
    } else {
        float x, y, z, w;
        asm volatile("ds_read_b32 %0, %4\n\tds_read_b32 %1, %4 offset:%5\n\tds_read_b32 %2, %4 offset:%6\n\tds_read_b32 %3, %4 offset:%7\n\ts_waitcnt lgkmcnt(0)"
                     : "=&v"(x), "=&v"(y), "=&v"(z), "=&v"(w) : "v"(at0), "n"(PITCH), "n"(2 * PITCH), "n"(3 * PITCH) : "memory");
        return typename El<T>::frag{x, y, z, w};
    }
}

// One product step: the fragments of the next step are requested, the products of this one are issued, and only then the
// requests are waited for, all in one block.  x: rows, w: outputs; nx, nw: the next step's.  The first s_nop covers an
// accumulator that was just written, settle() the products' own latency in front of anything that reads one.
#define NERF_BLOCK_HEAD "s_nop 1\n\t"
#define NERF_BLOCK_TAIL "s_waitcnt lgkmcnt(0)"
#define NERF_READ_X2 "ds_read_b128 %[nx0], %[pa]\n\tds_read_b128 %[nx1], %[pa] offset:4096\n\t"
#define NERF_READ_X1 "ds_read_b128 %[nx0], %[pa]\n\t"
#define NERF_READ_W2 "ds_read_b128 %[nw0], %[pb]\n\tds_read_b128 %[nw1], %[pb] offset:4096\n\t"
#define NERF_READ_W1 "ds_read_b128 %[nw0], %[pb]\n\t"
#define NERF_READ_TR(lo, hi, at) "ds_read_b64_tr_b16 %[" lo "], %[" at "]\n\tds_read_b64_tr_b16 %[" hi "], %[" at "] offset:%[rows4]\n\t"
#define NERF_MFMA(op, c, w, x) op " %[" c "], %[" w "], %[" x "], %[" c "]\n\t"
#define NERF_MFMA22(op) NERF_MFMA(op, "c00", "w0", "x0") NERF_MFMA(op, "c01", "w1", "x0") NERF_MFMA(op, "c10", "w0", "x1") NERF_MFMA(op, "c11", "w1", "x1")
#define NERF_MFMA21(op) NERF_MFMA(op, "c00", "w0", "x0") NERF_MFMA(op, "c10", "w0", "x1")
#define NERF_MFMA11(op) NERF_MFMA(op, "c00", "w0", "x0")

template <typename T, int MI, int NJ>
__device__ __forceinline__ void settle(f32x16 (&c)[MI][NJ]) {
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) asm volatile("s_nop 15\n\ts_nop 7" : "+v"(c[i][j]));
}

// 16-bit operands; OP names the instruction of the type
#define NERF_BLOCKS_16(T, OP)                                                                                                           \
    template <int MI, int NJ, typename F>                                                                                               \
    __device__ __forceinline__ void block_nt(T, f32x16 (&c)[MI][NJ], F (&x)[MI], F (&w)[NJ], unsigned pa, unsigned pb) {                \
        F nx[MI], nw[NJ];                                                                                                               \
        if constexpr (MI == 2 && NJ == 2)                                                                                               \
            asm volatile(NERF_BLOCK_HEAD NERF_READ_X2 NERF_READ_W2 NERF_MFMA22(OP) NERF_BLOCK_TAIL                                      \
                         : [c00] "+v"(c[0][0]), [c01] "+v"(c[0][1]), [c10] "+v"(c[1][0]), [c11] "+v"(c[1][1]), [nx0] "=&v"(nx[0]),      \
                           [nx1] "=&v"(nx[1]), [nw0] "=&v"(nw[0]), [nw1] "=&v"(nw[1])                                                   \
                         : [x0] "v"(x[0]), [x1] "v"(x[1]), [w0] "v"(w[0]), [w1] "v"(w[1]), [pa] "v"(pa), [pb] "v"(pb)                   \
                         : "memory");                                                                                                   \
        else if constexpr (MI == 2)                                                                                                     \
            asm volatile(NERF_BLOCK_HEAD NERF_READ_X2 NERF_READ_W1 NERF_MFMA21(OP) NERF_BLOCK_TAIL                                      \
                         : [c00] "+v"(c[0][0]), [c10] "+v"(c[1][0]), [nx0] "=&v"(nx[0]), [nx1] "=&v"(nx[1]), [nw0] "=&v"(nw[0])         \
                         : [x0] "v"(x[0]), [x1] "v"(x[1]), [w0] "v"(w[0]), [pa] "v"(pa), [pb] "v"(pb)                                   \
                         : "memory");                                                                                                   \
        else                                                                                                                            \
            asm volatile(NERF_BLOCK_HEAD NERF_READ_X1 NERF_READ_W1 NERF_MFMA11(OP) NERF_BLOCK_TAIL                                      \
                         : [c00] "+v"(c[0][0]), [nx0] "=&v"(nx[0]), [nw0] "=&v"(nw[0])                                                  \
                         : [x0] "v"(x[0]), [w0] "v"(w[0]), [pa] "v"(pa), [pb] "v"(pb)                                                   \
                         : "memory");                                                                                                   \
        for (int i = 0; i < MI; ++i) x[i] = nx[i];                                                                                      \
        for (int j = 0; j < NJ; ++j) w[j] = nw[j];                                                                                      \
    }                                                                                                                                   \
    template <int PITCH, int MI, int NJ, int NP, typename F>                                                                            \
    __device__ __forceinline__ void block_tr(T, f32x16 (&c)[MI][NJ], F (&x)[MI], F (&w)[NJ], unsigned pa, const unsigned (&pb)[NP],     \
                                             unsigned stage) {                                                                          \
        F nx[MI];                                                                                                                       \
        struct Two { s16x4 lo, hi; } nw[NJ];                                                                                            \
        if constexpr (MI == 2 && NJ == 2)                                                                                               \
            asm volatile(NERF_BLOCK_HEAD NERF_READ_X2 NERF_READ_TR("l0", "h0", "p0") NERF_READ_TR("l1", "h1", "p1") NERF_MFMA22(OP)     \
                         NERF_BLOCK_TAIL                                                                                                \
                         : [c00] "+v"(c[0][0]), [c01] "+v"(c[0][1]), [c10] "+v"(c[1][0]), [c11] "+v"(c[1][1]), [nx0] "=&v"(nx[0]),      \
                           [nx1] "=&v"(nx[1]), [l0] "=&v"(nw[0].lo), [h0] "=&v"(nw[0].hi), [l1] "=&v"(nw[1].lo), [h1] "=&v"(nw[1].hi)   \
                         : [x0] "v"(x[0]), [x1] "v"(x[1]), [w0] "v"(w[0]), [w1] "v"(w[1]), [pa] "v"(pa), [p0] "v"(pb[0] + stage),       \
                           [p1] "v"(pb[1] + stage), [rows4] "n"(4 * PITCH)                                                              \
                         : "memory");                                                                                                   \
        else if constexpr (MI == 2)                                                                                                     \
            asm volatile(NERF_BLOCK_HEAD NERF_READ_X2 NERF_READ_TR("l0", "h0", "p0") NERF_MFMA21(OP) NERF_BLOCK_TAIL                    \
                         : [c00] "+v"(c[0][0]), [c10] "+v"(c[1][0]), [nx0] "=&v"(nx[0]), [nx1] "=&v"(nx[1]), [l0] "=&v"(nw[0].lo),      \
                           [h0] "=&v"(nw[0].hi)                                                                                         \
                         : [x0] "v"(x[0]), [x1] "v"(x[1]), [w0] "v"(w[0]), [pa] "v"(pa), [p0] "v"(pb[0] + stage), [rows4] "n"(4 * PITCH) \
                         : "memory");                                                                                                   \
        else                                                                                                                            \
            asm volatile(NERF_BLOCK_HEAD NERF_READ_X1 NERF_READ_TR("l0", "h0", "p0") NERF_MFMA11(OP) NERF_BLOCK_TAIL                    \
                         : [c00] "+v"(c[0][0]), [nx0] "=&v"(nx[0]), [l0] "=&v"(nw[0].lo), [h0] "=&v"(nw[0].hi)                          \
                         : [x0] "v"(x[0]), [w0] "v"(w[0]), [pa] "v"(pa), [p0] "v"(pb[0] + stage), [rows4] "n"(4 * PITCH)                \
                         : "memory");                                                                                                   \
        for (int i = 0; i < MI; ++i) x[i] = nx[i];                                                                                      \
        for (int j = 0; j < NJ; ++j) w[j] = __builtin_bit_cast(F, nw[j]);                                                               \
    }
NERF_BLOCKS_16(__bf16, "v_mfma_f32_32x32x16_bf16")
NERF_BLOCKS_16(_Float16, "v_mfma_f32_32x32x16_f16")
#undef NERF_BLOCKS_16

// fp32: four products per fragment, alternating between the accumulators
#define NERF_OP32 "v_mfma_f32_32x32x2_f32"
#define NERF_MFMA32_1(e) NERF_MFMA(NERF_OP32, "c00", "w" e, "x" e)
#define NERF_MFMA32_2(e) NERF_MFMA(NERF_OP32, "c00", "w" e, "x" e) NERF_MFMA(NERF_OP32, "c10", "w" e, "y" e)
#define NERF_IN4(n, v) [n##0] "v"(v[0]), [n##1] "v"(v[1]), [n##2] "v"(v[2]), [n##3] "v"(v[3])
template <int MI, int NJ, typename F>
__device__ __forceinline__ void block_nt(float, f32x16 (&c)[MI][NJ], F (&x)[MI], F (&w)[NJ], unsigned pa, unsigned pb) {
    static_assert(NJ == 1, "fp32 tiles are one output tile wide per wave");
    F nx[MI], nw[NJ];
    if constexpr (MI == 2)
        asm volatile(NERF_BLOCK_HEAD NERF_READ_X2 NERF_READ_W1 NERF_MFMA32_2("0") NERF_MFMA32_2("1") NERF_MFMA32_2("2") NERF_MFMA32_2("3") NERF_BLOCK_TAIL
                     : [c00] "+v"(c[0][0]), [c10] "+v"(c[1][0]), [nx0] "=&v"(nx[0]), [nx1] "=&v"(nx[1]), [nw0] "=&v"(nw[0])
                     : NERF_IN4(x, x[0]), NERF_IN4(y, x[1]), NERF_IN4(w, w[0]), [pa] "v"(pa), [pb] "v"(pb)
                     : "memory");
    else
        asm volatile(NERF_BLOCK_HEAD NERF_READ_X1 NERF_READ_W1 NERF_MFMA32_1("0") NERF_MFMA32_1("1") NERF_MFMA32_1("2") NERF_MFMA32_1("3") NERF_BLOCK_TAIL
                     : [c00] "+v"(c[0][0]), [nx0] "=&v"(nx[0]), [nw0] "=&v"(nw[0])
                     : NERF_IN4(x, x[0]), NERF_IN4(w, w[0]), [pa] "v"(pa), [pb] "v"(pb)
                     : "memory");
    for (int i = 0; i < MI; ++i) x[i] = nx[i];
    w[0] = nw[0];
}
#define NERF_READ_B4 "ds_read_b32 %[n0], %[p0]\n\tds_read_b32 %[n1], %[p0] offset:%[row1]\n\tds_read_b32 %[n2], %[p0] offset:%[row2]\n\tds_read_b32 %[n3], %[p0] offset:%[row3]\n\t"
template <int PITCH, int MI, int NJ, int NP, typename F>
__device__ __forceinline__ void block_tr(float, f32x16 (&c)[MI][NJ], F (&x)[MI], F (&w)[NJ], unsigned pa, const unsigned (&pb)[NP], unsigned stage) {
    static_assert(NJ == 1 && NP == 1, "fp32 tiles are one output tile wide per wave");
    F nx[MI];
    float n0, n1, n2, n3;
    if constexpr (MI == 2)
        asm volatile(NERF_BLOCK_HEAD NERF_READ_X2 NERF_READ_B4 NERF_MFMA32_2("0") NERF_MFMA32_2("1") NERF_MFMA32_2("2") NERF_MFMA32_2("3") NERF_BLOCK_TAIL
                     : [c00] "+v"(c[0][0]), [c10] "+v"(c[1][0]), [nx0] "=&v"(nx[0]), [nx1] "=&v"(nx[1]), [n0] "=&v"(n0), [n1] "=&v"(n1),
                       [n2] "=&v"(n2), [n3] "=&v"(n3)
                     : NERF_IN4(x, x[0]), NERF_IN4(y, x[1]), NERF_IN4(w, w[0]), [pa] "v"(pa), [p0] "v"(pb[0] + stage), [row1] "n"(PITCH),
                       [row2] "n"(2 * PITCH), [row3] "n"(3 * PITCH)
                     : "memory");
    else
        asm volatile(NERF_BLOCK_HEAD NERF_READ_X1 NERF_READ_B4 NERF_MFMA32_1("0") NERF_MFMA32_1("1") NERF_MFMA32_1("2") NERF_MFMA32_1("3") NERF_BLOCK_TAIL
                     : [c00] "+v"(c[0][0]), [nx0] "=&v"(nx[0]), [n0] "=&v"(n0), [n1] "=&v"(n1), [n2] "=&v"(n2), [n3] "=&v"(n3)
                     : NERF_IN4(x, x[0]), NERF_IN4(w, w[0]), [pa] "v"(pa), [p0] "v"(pb[0] + stage), [row1] "n"(PITCH), [row2] "n"(2 * PITCH),
                       [row3] "n"(3 * PITCH)
                     : "memory");
    for (int i = 0; i < MI; ++i) x[i] = nx[i];
    w[0] = F{n0, n1, n2, n3};
}

template <typename T, bool WT, int BN>
__global__ __launch_bounds__(ST_THREADS) void stream_kernel(LinArgs p) {
    constexpr int E = piece<T>(), BK = step_len<T>(), WAVES = ST_THREADS / 64;
    constexpr int WM = BN == 64 ? 4 : 2, WO = WAVES / WM;                   // waves along rows and outputs
    constexpr int MI = TILE_ROWS / WM / 32, NJ = BN / WO / 32;
    constexpr int A_BYTES = TILE_ROWS * 128, B_BYTES = WT ? tr_bytes<T, BN>() : BN * 128, STAGE = A_BYTES + B_BYTES;
    constexpr int NA = A_BYTES / 1024 / WAVES, NB = B_BYTES / 1024 / WAVES; // copies of a wave per step
    constexpr int COPIES = NA + NB;
    constexpr int ITEMS = st_items<BN>();
    constexpr int STORES = MI * NJ * (sizeof(T) == 2 ? 2 : 4);              // stores of a wave per item
    static_assert(COPIES + 2 * STORES < 64, "vmcnt counts to 63");
    __shared__ __attribute__((aligned(1024))) char lds[3 * STAGE];
    __shared__ int row_tab[ITEMS][TILE_ROWS];
    __shared__ __attribute__((aligned(16))) T bias_tab[ITEMS][BN];
    __shared__ int d_grp[ITEMS], d_o0[ITEMS], d_cnt[ITEMS], d_pos[ITEMS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m_off = (wave % WM) * (MI * 32), o_off = (wave / WM) * (NJ * 32);
    const int G = p.rows.n_groups, O = p.O, C = p.C;
    const int nk = (C + BK - 1) / BK;
    T* out = (T*)p.out;
    const float least = p.relu ? 0.0f : -__builtin_inff();
    const unsigned bits = p.relu ? 0x7fffffffu : 0xffffffffu;
    typedef __attribute__((address_space(3))) char* lds_ptr;
    const unsigned lds0 = (unsigned)(uintptr_t)(lds_ptr)lds, rows0 = (unsigned)(uintptr_t)(lds_ptr)row_tab, bias0 = (unsigned)(uintptr_t)(lds_ptr)bias_tab;

    // An XCD takes a run of consecutive items and deals them to its workgroups in turn, so that the output tiles of the same
    // rows are worked on at the same time and the rows come from memory once (in runs per workgroup, 1024 outputs of 65 536
    // rows fetched the rows four times).
    const Tables tables(p.rows, lane);
    const int64_t work = (int64_t)tables.total * p.tiles_o, xcd = blockIdx.x & 7;
    const int64_t begin = work * xcd / 8 + (blockIdx.x >> 3), finish = work * (xcd + 1) / 8, stride = gridDim.x >> 3;

    // Copy i of wave w fills LDS slots (w n + i) 64 + lane of its tile; the lane picks the row and the piece that belong there.
    int a_row[NA], a_q[NA], b_row[NB], b_q[NB];
#pragma unroll
    for (int i = 0; i < NA; ++i) {
        const int slot = (wave * NA + i) * 64 + lane;
        a_row[i] = slot >> 3;
        a_q[i] = (slot & 7) ^ ((a_row[i] >> 1) & 7);
    }
    constexpr int BPR = BN / E;                                             // pieces per row of a transposed W tile
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        const int slot = (wave * NB + i) * 64 + lane;
        b_row[i] = WT ? slot / BPR : slot >> 3;
        b_q[i] = WT ? (slot % BPR) ^ tr_swap<T, BN>(b_row[i]) : (slot & 7) ^ ((b_row[i] >> 1) & 7);
    }
    // LDS addresses of this lane's fragments within a stage, by product step
    unsigned fa[ROW_PIECES / 2], fb[ROW_PIECES / 2][WT ? NJ : 1];
#pragma unroll
    for (int s = 0; s < ROW_PIECES / 2; ++s) {
        fa[s] = lds0 + nt_addr(m_off + (lane & 31), 2 * s + (lane >> 5));
        if constexpr (!WT) {
            fb[s][0] = lds0 + A_BYTES + nt_addr(o_off + (lane & 31), 2 * s + (lane >> 5));
        } else {
#pragma unroll
            for (int j = 0; j < NJ; ++j) fb[s][j] = lds0 + A_BYTES + tr_lane<T, BN>(o_off + 32 * j, s, lane);
        }
    }

    for (int64_t first = begin; first < finish; first += ITEMS * stride) {
        const int64_t left = (finish - first + stride - 1) / stride;
        const int items = (int)(left < ITEMS ? left : ITEMS);
        __syncthreads();
        for (int i = wave; i < items; i += WAVES) {
            const Tile t = tables.tile(p.rows, first + i * stride, p.tiles_o, BN);
            if (lane == 0) { d_grp[i] = t.group; d_o0[i] = t.o0; d_cnt[i] = t.count; d_pos[i] = (int)t.pos0; }
        }
        __syncthreads();
#pragma unroll 3
        for (int j = tid; j < items * TILE_ROWS; j += ST_THREADS) {
            const int i = j / TILE_ROWS, row = p.rows.order[d_pos[i] + min(j % TILE_ROWS, d_cnt[i] - 1)];
            row_tab[0][j] = min(max(row, 0), (int)p.rows.n - 1);
        }
        if (p.bias) {
#pragma unroll 3
            for (int j = tid; j < items * BN; j += ST_THREADS) {
                const int i = j / BN, o = d_o0[i] + j % BN, g = min(d_grp[i], G - 1);
                bias_tab[0][j] = ((const T*)p.bias)[(int64_t)g * O + out_of<E>(o, O)];
            }
        } else {
            for (int j = tid; j < items * BN; j += ST_THREADS) bias_tab[0][j] = (T)0.0f;
        }
        __syncthreads();
        int real = items;                                                   // the rows of no group come last
        while (real > 0 && d_grp[real - 1] == G) --real;
        for (int i = real; i < items; ++i) {
            const int o0 = d_o0[i], pieces = ((O - o0 < BN ? O - o0 : BN) + E - 1) / E;
            Pack<T, E> zero;
#pragma unroll
            for (int e = 0; e < E; ++e) zero.v[e] = (T)0.0f;
            for (int j = tid; j < d_cnt[i] * pieces; j += ST_THREADS)
                store_any<T, E>(out + (int64_t)row_tab[i][j / pieces] * O + out_of<E>(o0 + (j % pieces) * E, O), zero);
        }
        const int steps = real * nk;
        if (steps == 0) continue;

        // ---- copies: step c_k of item c_item into buffer c_buf ----
        int c_item = 0, c_k = 0, c_buf = 0;
        const T *pa[NA], *pb[NB];
        auto copy_step = [&]() {
            if (c_k == 0) {
                const int g = min(__builtin_amdgcn_readfirstlane(lds_int((unsigned)(uintptr_t)(lds_ptr)&d_grp[c_item])), G - 1);
                const int o0 = __builtin_amdgcn_readfirstlane(lds_int((unsigned)(uintptr_t)(lds_ptr)&d_o0[c_item]));
#pragma unroll
                for (int i = 0; i < NA; ++i) {
                    const int64_t row = lds_int(rows0 + (c_item * TILE_ROWS + a_row[i]) * 4);
                    pa[i] = (const T*)p.a + row * p.a_ld + a_q[i] * E;
                }
                const T* w = (const T*)p.w + g * p.w_gs;
#pragma unroll
                for (int i = 0; i < NB; ++i) {
                    if constexpr (WT) {
                        const int o = o0 + b_q[i] * E;
                        pb[i] = w + b_row[i] * p.w_ld + (o < p.w_ld ? o : p.w_ld - E);
                    } else {
                        pb[i] = w + out_of<E>(o0 + b_row[i], O) * p.w_ld + b_q[i] * E;
                    }
                }
            }
            char* const to = lds + c_buf * STAGE + wave * (NA * 1024);
            char* const to_b = lds + c_buf * STAGE + A_BYTES + wave * (NB * 1024);
            const int k0 = c_k * BK;
            if (k0 + BK <= (WT ? p.w_rows : C)) {
#pragma unroll
                for (int i = 0; i < NA; ++i) copy_piece(pa[i], to + i * 1024);
#pragma unroll
                for (int i = 0; i < NB; ++i) copy_piece(pb[i], to_b + i * 1024);
            } else {                                                        // what lies behind the sum is read as zero
#pragma unroll
                for (int i = 0; i < NA; ++i) copy_piece(k0 + a_q[i] * E < C ? (const void*)pa[i] : (const void*)&ZERO_PIECE, to + i * 1024);
#pragma unroll
                for (int i = 0; i < NB; ++i)
                    copy_piece((WT ? k0 + b_row[i] < p.w_rows : k0 + b_q[i] * E < C) ? (const void*)pb[i] : (const void*)&ZERO_PIECE, to_b + i * 1024);
            }
            if (c_item * nk + c_k + 1 < steps) {
#pragma unroll
                for (int i = 0; i < NA; ++i) pa[i] += BK;
#pragma unroll
                for (int i = 0; i < NB; ++i) pb[i] += WT ? BK * p.w_ld : BK;
            }
            // behind the last step the last one is copied again, into a buffer that nothing reads any more
            if (c_item * nk + c_k + 1 < steps && ++c_k == nk) { c_k = 0; ++c_item; }
            c_buf = c_buf == 2 ? 0 : c_buf + 1;
        };
        f32x16 acc[MI][NJ];
        auto clear = [&]() {
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NJ; ++j)
#pragma unroll
                    for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
        };
        auto finish_item = [&](int item) {
            const int o0 = __builtin_amdgcn_readfirstlane(lds_int((unsigned)(uintptr_t)(lds_ptr)&d_o0[item])) + o_off;
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                const int64_t row = lds_int(rows0 + (item * TILE_ROWS + m_off + 32 * i + (lane & 31)) * 4);
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    float z[16];
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        const unsigned at = bias0 + (item * BN + o_off + 32 * j + 8 * h + 4 * (lane >> 5)) * (int)sizeof(T);
                        float b[4];
                        if constexpr (sizeof(T) == 2) {
                            uint2 v;
                            asm volatile("ds_read_b64 %0, %1\n\ts_waitcnt lgkmcnt(0)" : "=&v"(v) : "v"(at) : "memory");
                            const Pack<T, 4> q = __builtin_bit_cast(Pack<T, 4>, v);
#pragma unroll
                            for (int e = 0; e < 4; ++e) b[e] = (float)q.v[e];
                        } else {
                            const f32x4 q = lds_quad(at);
#pragma unroll
                            for (int e = 0; e < 4; ++e) b[e] = q[e];
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float v = acc[i][j][4 * h + e] + b[e];
                            z[4 * h + e] = relu_or_not(v, least, bits);
                        }
                    }
                    if constexpr (sizeof(T) == 2) {
#pragma unroll
                        for (int h = 0; h < 4; h += 2) {
                            unsigned x[2], y[2];
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                Pack<T, 2> u, v;
                                u.v[0] = (T)z[4 * h + 2 * e]; u.v[1] = (T)z[4 * h + 2 * e + 1];
                                v.v[0] = (T)z[4 * h + 4 + 2 * e]; v.v[1] = (T)z[4 * h + 4 + 2 * e + 1];
                                const auto sw = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, u), __builtin_bit_cast(unsigned, v), false, false);
                                x[e] = sw[0];
                                y[e] = sw[1];
                            }
                            const uint4 q = make_uint4(x[0], x[1], y[0], y[1]);
                            store_any<T, E>(out + row * O + out_of<E>(o0 + 32 * j + 8 * h + 8 * (lane >> 5), O), __builtin_bit_cast(Pack<T, E>, q));
                        }
                    } else {
#pragma unroll
                        for (int h = 0; h < 4; ++h) {
                            const float4 q = make_float4(z[4 * h], z[4 * h + 1], z[4 * h + 2], z[4 * h + 3]);
                            store_any<T, E>(out + row * O + out_of<E>(o0 + 32 * j + 8 * h + 4 * (lane >> 5), O), __builtin_bit_cast(Pack<T, E>, q));
                        }
                    }
                }
            }
        };

        wait_copies<0>();                                                   // stores of the last round of items
        clear();
        int item = 0, k = 0, buf = 0, late = 0;                             // late: bit 0 / 1: stores behind the newest / the other copies
        auto wait_step = [&]() {
            if (late == 0) wait_copies<COPIES>();
            else if (late == 3) wait_copies<COPIES + 2 * STORES>();
            else wait_copies<COPIES + STORES>();
            __builtin_amdgcn_s_barrier();
            late = (late << 1) & 3;
        };
        auto end_step = [&]() {
            if (++k == nk) {
                settle<T, MI, NJ>(acc);
                finish_item(item);
                clear();
                k = 0;
                ++item;
                late |= 1;
            }
        };
        copy_step();
        copy_step();
        copy_step();
        // The last fragments of a step are in registers one product step before its end: there the barrier frees its buffer for
        // step s + 3 and the first fragments of step s + 1 are requested.
        constexpr int S = ROW_PIECES / 2;
        typename El<T>::frag fx[MI], fw[NJ];
        wait_copies<2 * COPIES>();
        __builtin_amdgcn_s_barrier();
        if constexpr (!WT) {
            read_nt<typename El<T>::frag, MI, NJ>(fx, fw, fa[0], fb[0][0]);
        } else {
            read_rows<typename El<T>::frag, MI>(fx, fa[0]);
#pragma unroll
            for (int j = 0; j < NJ; ++j) fw[j] = read_tr<T, BN * (int)sizeof(T)>(fb[0][j]);
        }
        for (int s = 0; s < steps; ++s) {
#pragma unroll
            for (int u = 0; u < S; ++u) {
                unsigned stage = buf * STAGE;
                if (u == S - 1) {
                    wait_step();
                    buf = buf == 2 ? 0 : buf + 1;
                    stage = buf * STAGE;
                }
                const int n = (u + 1) % S;
                if constexpr (!WT) block_nt<MI, NJ>(T(), acc, fx, fw, fa[n] + stage, fb[n][0] + stage);
                else block_tr<BN * (int)sizeof(T)>(T(), acc, fx, fw, fa[n] + stage, fb[n], stage);
            }
            copy_step();                                                    // beside the last products
            end_step();
        }
        wait_copies<0>();                                                   // nothing may land once the rows are written anew
    }
}

// ---- through registers: any row length, any alignment ------------------------------------------------------------
// The same product, one workgroup of four waves per tile of 128 rows x BN outputs; a step is requested before the products of
// the one before it (65 536 rows, 67 -> 256 bf16: forward 24 us, 28 with a bias; in whole pieces, 64 -> 256, 18).
template <typename T, bool WT, int BN>
__global__ __launch_bounds__(THREADS, 2) void linear_kernel(LinArgs p) {
    constexpr int E = piece<T>(), BK = step_len<T>();
    constexpr int A_BYTES = TILE_ROWS * 128;
    constexpr int B_BYTES = WT ? tr_bytes<T, BN>() : BN * 128;
    constexpr int PITCH = BN * 2 + 16;                                      // 16-bit output tile in LDS
    constexpr int LDS = sizeof(T) == 2 && TILE_ROWS * PITCH > A_BYTES + B_BYTES ? TILE_ROWS * PITCH : A_BYTES + B_BYTES;
    __shared__ __attribute__((aligned(16))) char lds[LDS];
    __shared__ int row_of[TILE_ROWS];
    constexpr int MI = BN == 128 ? 2 : 1, NJ = 2;                           // 32-row and 32-output tiles of a wave
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int m_off = BN == 128 ? (wave & 1) * 64 : wave * 32, o_off = BN == 128 ? (wave >> 1) * 64 : 0;

    // consecutive tiles on one XCD (workgroups go round the eight XCDs), output tiles of the same rows next to each other
    const Tables tables(p.rows, lane);
    const int64_t work = (int64_t)tables.total * p.tiles_o;
    const int64_t per_xcd = (work + 7) / 8, local = (blockIdx.x >> 3) + (int64_t)blockIdx.y * p.grid_row;
    const int64_t at = (blockIdx.x & 7) * per_xcd + local;
    if (local >= per_xcd || at >= work) return;
    const Tile t = tables.tile(p.rows, at, p.tiles_o, BN);
    const int g = t.group, o0 = t.o0;
    if (tid < TILE_ROWS) row_of[tid] = tid < t.count ? row_at(p.rows, t.pos0 + tid) : -1;
    __syncthreads();
    T* out = (T*)p.out;
    const int O = p.O, C = p.C;
    if (g == p.rows.n_groups) {                                             // rows of no group
        const int width = O - o0 < BN ? O - o0 : BN;
        for (int i = tid; i < t.count * width; i += THREADS) {
            const int row = row_of[i / width];
            if (row >= 0) out[(int64_t)row * O + o0 + i % width] = (T)0.0f;
        }
        return;
    }
    const T* w = (const T*)p.w + (int64_t)g * O * C;
    char* const A = lds;
    char* const B = lds + A_BYTES;
    constexpr int BPR = BN / E;                                             // pieces per row of a transposed W tile
    constexpr int NA = TILE_ROWS * 8 / THREADS, NB = B_BYTES / 16 / THREADS;
    const int q = tid & 7, r0 = tid >> 3;
    int rows[NA];
#pragma unroll
    for (int i = 0; i < NA; ++i) rows[i] = row_of[r0 + 32 * i];
    Pack<T, E> ra[NA], rb[NB];
    auto fill = [&](int k0) {
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            const int64_t row = rows[i] < 0 ? 0 : rows[i];
            ra[i] = load_piece<T>((const T*)p.a + row * p.a_ld, k0 + q * E, C, rows[i] >= 0);
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            if constexpr (WT) {
                const int c = k0 + (tid + i * THREADS) / BPR;
                rb[i] = load_piece<T>(w + (int64_t)(c < C ? c : 0) * O, o0 + (tid + i * THREADS) % BPR * E, O, c < C);
            } else {
                const int o = o0 + r0 + 32 * i;
                rb[i] = load_piece<T>(w + (int64_t)(o < O ? o : 0) * C, k0 + q * E, C, o < O);
            }
        }
    };
    f32x16 acc[MI][NJ];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    fill(0);
    for (int k0 = 0; k0 < C; k0 += BK) {
#pragma unroll
        for (int i = 0; i < NA; ++i) put_piece<T, E>(A + nt_addr(r0 + 32 * i, q), ra[i]);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            if constexpr (WT) put_piece<T, E>(B + tr_addr<T, BN>((tid + i * THREADS) / BPR, (tid + i * THREADS) % BPR), rb[i]);
            else put_piece<T, E>(B + nt_addr(r0 + 32 * i, q), rb[i]);
        }
        __syncthreads();
        if (k0 + BK < C) fill(k0 + BK);
#pragma unroll
        for (int s = 0; s < ROW_PIECES / 2; ++s) {
            typename El<T>::frag fx[MI], fw[NJ];
#pragma unroll
            for (int i = 0; i < MI; ++i) fx[i] = nt_frag<T>(A, m_off + 32 * i, s, lane);
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                if constexpr (WT) fw[j] = tr_frag<T, BN>(B, o_off + 32 * j, s, lane);
                else fw[j] = nt_frag<T>(B, o_off + 32 * j, s, lane);
            }
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NJ; ++j) acc[i][j] = El<T>::mfma(fw[j], fx[i], acc[i][j]);
        }
        __syncthreads();                                                    // every wave has read the step
    }

    // bias, ReLU, and the rows back to where they belong
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            const int o = o0 + o_off + 32 * j + 8 * h + 4 * (lane >> 5);
            float b[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (p.bias)
#pragma unroll
                for (int e = 0; e < 4; ++e) b[e] = o + e < O ? (float)((const T*)p.bias)[(int64_t)g * O + o + e] : 0.0f;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float z = acc[i][j][4 * h + e] + b[e];
                    if (p.relu) z = z < 0.0f ? 0.0f : fabsf(z);             // keeps a NaN, without its sign
                    acc[i][j][4 * h + e] = z;
                }
        }
    if constexpr (sizeof(T) == 2) {
        // through LDS, so that a wave stores neighbouring outputs of a row together
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
            const int at = tid + i * THREADS, m = at / (BN / E), c = at % (BN / E) * E, row = row_of[m];
            if (row < 0 || o0 + c >= O) continue;
            put_row_piece<T>(out + (int64_t)row * O, o0 + c, O, *reinterpret_cast<const Pack<T, E>*>(lds + m * PITCH + c * 2));
        }
    } else {
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            const int row = row_of[m_off + 32 * i + (lane & 31)];
            if (row < 0) continue;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int o = o0 + o_off + 32 * j + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
                    if (o < O) out[(int64_t)row * O + o] = (T)acc[i][j][r];
                }
        }
    }
}

struct WgradArgs {
    Rows rows;
    int K, N, tiles_k, tiles_n;
    int Kp, Np;                      // columns of x and dy that can be read (streaming form: whole pieces)
    int chunk;                       // tiles of one workgroup
    int64_t x_ld, dy_ld;
    const void *x, *dy;
    void *dw, *db;
    float *part_w, *part_b;          // [2 * chunks][N * K], [2 * chunks][N]: slot 2c a group that came in from the left of
};                                   // chunk c, slot 2c + 1 one that began in it and goes on to the right

// dW[n][k] = sum over rows dZ[row][n] x[row][k], streaming form.  A workgroup of eight waves owns one BD x BX block of every
// dW it meets and walks `chunk` consecutive tiles of the flat tile list, whatever groups they belong to, so all workgroups
// have equal work however uneven the groups are.  A group that lies inside one chunk is finished here; the pieces of a longer
// one go to the workspace and are added up in order by wgrad_join_kernel (no atomics: the result does not depend on timing).
//
// Rows of both operands are copied as they are into a ring of three LDS buffers,
// as in stream_kernel; a row behind the end of a tile is read from a piece of zeros.  The sum of dZ over the rows comes from
// the fragments: the four waves that share a range of n take one product step of four each.
constexpr int WG_TILES = 24;            // tiles whose rows are in LDS at a time

#define NERF_WG_BLOCK(T, OP)                                                                                                            \
    template <int PD, int PX, int NJ, typename F>                                                                                       \
    __device__ __forceinline__ void block_wgrad(T, f32x16 (&c)[2][NJ], F (&d)[2], F (&x)[NJ], unsigned d0, unsigned d1, unsigned x0,    \
                                                unsigned x1) {                                                                          \
        struct Two { s16x4 lo, hi; } nd[2], nx[NJ];                                                                                     \
        if constexpr (NJ == 2)                                                                                                          \
            asm volatile(NERF_BLOCK_HEAD NERF_READ_TRD("l0", "h0", "d0") NERF_READ_TRX("l2", "h2", "x0") NERF_READ_TRD("l1", "h1", "d1") \
                         NERF_READ_TRX("l3", "h3", "x1") NERF_MFMA(OP, "c00", "e0", "f0") NERF_MFMA(OP, "c01", "e0", "f1")              \
                         NERF_MFMA(OP, "c10", "e1", "f0") NERF_MFMA(OP, "c11", "e1", "f1") NERF_BLOCK_TAIL                              \
                         : [c00] "+v"(c[0][0]), [c01] "+v"(c[0][1]), [c10] "+v"(c[1][0]), [c11] "+v"(c[1][1]), [l0] "=&v"(nd[0].lo),    \
                           [h0] "=&v"(nd[0].hi), [l1] "=&v"(nd[1].lo), [h1] "=&v"(nd[1].hi), [l2] "=&v"(nx[0].lo), [h2] "=&v"(nx[0].hi), \
                           [l3] "=&v"(nx[1].lo), [h3] "=&v"(nx[1].hi)                                                                   \
                         : [e0] "v"(d[0]), [e1] "v"(d[1]), [f0] "v"(x[0]), [f1] "v"(x[1]), [d0] "v"(d0), [d1] "v"(d1), [x0] "v"(x0),    \
                           [x1] "v"(x1), [rowsd] "n"(4 * PD), [rowsx] "n"(4 * PX)                                                       \
                         : "memory");                                                                                                   \
        else                                                                                                                            \
            asm volatile(NERF_BLOCK_HEAD NERF_READ_TRD("l0", "h0", "d0") NERF_READ_TRX("l2", "h2", "x0") NERF_READ_TRD("l1", "h1", "d1") \
                         NERF_MFMA(OP, "c00", "e0", "f0") NERF_MFMA(OP, "c10", "e1", "f0") NERF_BLOCK_TAIL                              \
                         : [c00] "+v"(c[0][0]), [c10] "+v"(c[1][0]), [l0] "=&v"(nd[0].lo), [h0] "=&v"(nd[0].hi), [l1] "=&v"(nd[1].lo),  \
                           [h1] "=&v"(nd[1].hi), [l2] "=&v"(nx[0].lo), [h2] "=&v"(nx[0].hi)                                             \
                         : [e0] "v"(d[0]), [e1] "v"(d[1]), [f0] "v"(x[0]), [d0] "v"(d0), [d1] "v"(d1), [x0] "v"(x0),                    \
                           [rowsd] "n"(4 * PD), [rowsx] "n"(4 * PX)                                                                     \
                         : "memory");                                                                                                   \
        for (int i = 0; i < 2; ++i) d[i] = __builtin_bit_cast(F, nd[i]);                                                                \
        for (int j = 0; j < NJ; ++j) x[j] = __builtin_bit_cast(F, nx[j]);                                                               \
    }
#define NERF_READ_TRD(lo, hi, at) "ds_read_b64_tr_b16 %[" lo "], %[" at "]\n\tds_read_b64_tr_b16 %[" hi "], %[" at "] offset:%[rowsd]\n\t"
#define NERF_READ_TRX(lo, hi, at) "ds_read_b64_tr_b16 %[" lo "], %[" at "]\n\tds_read_b64_tr_b16 %[" hi "], %[" at "] offset:%[rowsx]\n\t"
NERF_WG_BLOCK(__bf16, "v_mfma_f32_32x32x16_bf16")
NERF_WG_BLOCK(_Float16, "v_mfma_f32_32x32x16_f16")
#undef NERF_WG_BLOCK

// fp32: one block per 32 x 32 sums, four products each
#define NERF_READ_F4(n, at) "ds_read_b32 %[" n "0], %[" at "]\n\tds_read_b32 %[" n "1], %[" at "] offset:%[row1]\n\tds_read_b32 %[" n "2], %[" at "] offset:%[row2]\n\tds_read_b32 %[" n "3], %[" at "] offset:%[row3]\n\t"
#define NERF_MFMA32_W NERF_MFMA(NERF_OP32, "c", "e0", "f0") NERF_MFMA(NERF_OP32, "c", "e1", "f1") NERF_MFMA(NERF_OP32, "c", "e2", "f2") NERF_MFMA(NERF_OP32, "c", "e3", "f3")
template <int PD, int PX, int NJ, typename F>
__device__ __forceinline__ void block_wgrad(float, f32x16 (&c)[2][NJ], F (&d)[2], F (&x)[NJ], unsigned d0, unsigned d1, unsigned x0, unsigned) {
    static_assert(NJ == 1 && PD == PX, "fp32 blocks are 128 x 128");
    float a[4], b[4], w[4];
    asm volatile(NERF_BLOCK_HEAD NERF_READ_F4("n", "at") NERF_READ_F4("m", "to") NERF_MFMA32_W NERF_BLOCK_TAIL
                 : [c] "+v"(c[0][0]), [n0] "=&v"(a[0]), [n1] "=&v"(a[1]), [n2] "=&v"(a[2]), [n3] "=&v"(a[3]), [m0] "=&v"(w[0]), [m1] "=&v"(w[1]),
                   [m2] "=&v"(w[2]), [m3] "=&v"(w[3])
                 : NERF_IN4(e, d[0]), NERF_IN4(f, x[0]), [at] "v"(d0), [to] "v"(x0), [row1] "n"(PD), [row2] "n"(2 * PD), [row3] "n"(3 * PD)
                 : "memory");
    asm volatile(NERF_BLOCK_HEAD NERF_READ_F4("n", "at") NERF_MFMA32_W NERF_BLOCK_TAIL
                 : [c] "+v"(c[1][0]), [n0] "=&v"(b[0]), [n1] "=&v"(b[1]), [n2] "=&v"(b[2]), [n3] "=&v"(b[3])
                 : NERF_IN4(e, d[1]), NERF_IN4(f, x[0]), [at] "v"(d1), [row1] "n"(PD), [row2] "n"(2 * PD), [row3] "n"(3 * PD)
                 : "memory");
    d[0] = F{a[0], a[1], a[2], a[3]};
    d[1] = F{b[0], b[1], b[2], b[3]};
    x[0] = F{w[0], w[1], w[2], w[3]};
}

template <typename T, int BX>
__global__ __launch_bounds__(ST_THREADS) void wgrad_stream_kernel(WgradArgs p) {
    constexpr int E = piece<T>(), BK = step_len<T>(), WAVES = ST_THREADS / 64, BD = 128;
    constexpr int PER_TILE = TILE_ROWS / BK, S = ROW_PIECES / 2;
    constexpr int MI = 2, NJ = BX / 4 / 32;                                 // waves: 2 along n, 4 along k
    constexpr int D_BYTES = tr_bytes<T, BD>(), X_BYTES = tr_bytes<T, BX>(), STAGE = D_BYTES + X_BYTES;
    constexpr int ND = D_BYTES / 1024 / WAVES, NX = X_BYTES / 1024 / WAVES;
    constexpr int COPIES = ND + NX;
    constexpr int DPR = BD / E, XPR = BX / E;                               // pieces of a row
    __shared__ __attribute__((aligned(1024))) char lds[3 * STAGE];
    __shared__ int row_tab[WG_TILES][TILE_ROWS];
    __shared__ int tile_pos[WG_TILES], tile_cnt[WG_TILES], tile_grp[WG_TILES + 1];
    __shared__ float red[4][BD];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n_off = (wave & 1) * 64, wk = wave >> 1, k_off = wk * (BX / 4);
    typedef __attribute__((address_space(3))) char* lds_ptr;
    const unsigned lds0 = (unsigned)(uintptr_t)(lds_ptr)lds, rows0 = (unsigned)(uintptr_t)(lds_ptr)row_tab, grp0 = (unsigned)(uintptr_t)(lds_ptr)tile_grp;

    // the blocks of one chunk next to each other, on one XCD where there are eight chunks or more: they read the same rows
    const int G = p.rows.n_groups, K = p.K, N = p.N;
    const int tiles = grp::checked_tiles(p.rows.tile_base[G], p.rows.most_tiles);      // the rows of no group stay out
    const int blocks = p.tiles_n * p.tiles_k;
    const int64_t chunks = (tiles + p.chunk - 1) / p.chunk;
    const int64_t per_xcd = (chunks * blocks + 7) / 8, local = blockIdx.x >> 3;
    const int64_t at = (blockIdx.x & 7) * per_xcd + local;
    if (local >= per_xcd || at >= chunks * blocks) return;
    const int c = (int)(at / blocks), blk = (int)(at % blocks);
    const int n0 = (blk / p.tiles_k) * BD, k0 = (blk % p.tiles_k) * BX;
    const int t0 = c * p.chunk, t1 = t0 + p.chunk < tiles ? t0 + p.chunk : tiles;

    int d_row[ND], x_row[NX];
    int64_t d_col[ND], x_col[NX];
#pragma unroll
    for (int i = 0; i < ND; ++i) {
        const int slot = (wave * ND + i) * 64 + lane;
        d_row[i] = slot / DPR;
        const int col = n0 + ((slot % DPR) ^ tr_swap<T, BD>(d_row[i])) * E;
        d_col[i] = col < p.Np ? col : p.Np - E;                             // columns behind the last are not stored
    }
#pragma unroll
    for (int i = 0; i < NX; ++i) {
        const int slot = (wave * NX + i) * 64 + lane;
        x_row[i] = slot / XPR;
        const int col = k0 + ((slot % XPR) ^ tr_swap<T, BX>(x_row[i])) * E;
        x_col[i] = col < p.Kp ? col : p.Kp - E;
    }
    unsigned fd[S][MI], fx[S][NJ];
#pragma unroll
    for (int s = 0; s < S; ++s) {
#pragma unroll
        for (int i = 0; i < MI; ++i) fd[s][i] = lds0 + tr_lane<T, BD>(n_off + 32 * i, s, lane);
#pragma unroll
        for (int j = 0; j < NJ; ++j) fx[s][j] = lds0 + D_BYTES + tr_lane<T, BX>(k_off + 32 * j, s, lane);
    }
    f32x16 acc[MI][NJ];
    float sum[MI];                                                          // of dZ over this lane's rows
    auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            sum[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
        }
    };
    const bool bias = p.db && k0 == 0;
    auto flush = [&](int g) {
        // within [0, tiles], so that a single chunk, which has no workspace, finishes every group
        const int b0 = grp::checked_tiles(p.rows.tile_base[g], tiles), b1 = grp::checked_tiles(p.rows.tile_base[g + 1], tiles);
        const bool whole = b0 >= t0 && b1 <= t1;
        const int64_t slot = 2 * (int64_t)c + (b0 >= t0 ? 1 : 0);
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int n = n0 + n_off + 32 * i + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
                if (n >= N) continue;
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    const int k = k0 + k_off + 32 * j + (lane & 31);
                    if (k >= K) continue;
                    if (whole) ((T*)p.dw)[((int64_t)g * N + n) * K + k] = (T)acc[i][j][r];
                    else p.part_w[(slot * N + n) * K + k] = acc[i][j][r];
                }
            }
        if (bias) {
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                const float v = sum[i] + __shfl_xor(sum[i], 32, 64);
                if (lane < 32) red[wk][n_off + 32 * i + lane] = v;
            }
            __syncthreads();
            if (tid < BD && n0 + tid < N) {
                const float v = (red[0][tid] + red[1][tid]) + (red[2][tid] + red[3][tid]);
                if (whole) ((T*)p.db)[(int64_t)g * N + n0 + tid] = (T)v;
                else p.part_b[slot * N + n0 + tid] = v;
            }
            __syncthreads();
        }
        wait_copies<0>();                                                   // the counts of the steps to come have no stores in them
    };
    clear();

    for (int first = t0; first < t1; first += WG_TILES) {
        const int here = t1 - first < WG_TILES ? t1 - first : WG_TILES;
        __syncthreads();
        for (int i = tid; i <= here; i += ST_THREADS) {
            const int t = first + i;
            int lo = 0, hi = G;                                             // last group with tile_base <= t
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (p.rows.tile_base[mid] <= t) lo = mid;
                else hi = mid;
            }
            tile_grp[i] = t < t1 ? lo : -1;                                 // of the tile behind the last one here too
            if (i < here) {
                const grp::Span span = grp::checked_span(p.rows.offsets[lo] + ((int64_t)t - p.rows.tile_base[lo]) * TILE_ROWS, p.rows.offsets[lo + 1], p.rows.n);
                tile_pos[i] = (int)span.pos;
                tile_cnt[i] = span.count;
            }
        }
        __syncthreads();
#pragma unroll 3
        for (int j = tid; j < here * TILE_ROWS; j += ST_THREADS) {
            const int i = j / TILE_ROWS, r = j % TILE_ROWS, cnt = tile_cnt[i];
            const int row = p.rows.order[tile_pos[i] + (r < cnt ? r : 0)];
            row_tab[0][j] = r < cnt && row >= 0 && row < p.rows.n ? row : -1;
        }
        __syncthreads();
        const int steps = here * PER_TILE;
        int c_step = 0, c_buf = 0;
        auto copy_step = [&]() {
            char* const to = lds + c_buf * STAGE;
            const unsigned rows = rows0 + c_step * (BK * 4);
            int rd[ND], rx[NX];
            if constexpr (ND == 2 && NX == 4)
                asm volatile("ds_read_b32 %0, %6\n\tds_read_b32 %1, %7\n\tds_read_b32 %2, %8\n\tds_read_b32 %3, %9\n\tds_read_b32 %4, %10\n\tds_read_b32 %5, %11\n\ts_waitcnt lgkmcnt(0)"
                             : "=&v"(rd[0]), "=&v"(rd[1]), "=&v"(rx[0]), "=&v"(rx[1]), "=&v"(rx[2]), "=&v"(rx[3])
                             : "v"(rows + d_row[0] * 4), "v"(rows + d_row[1] * 4), "v"(rows + x_row[0] * 4), "v"(rows + x_row[1] * 4),
                               "v"(rows + x_row[2] * 4), "v"(rows + x_row[3] * 4) : "memory");
            else
                asm volatile("ds_read_b32 %0, %4\n\tds_read_b32 %1, %5\n\tds_read_b32 %2, %6\n\tds_read_b32 %3, %7\n\ts_waitcnt lgkmcnt(0)"
                             : "=&v"(rd[0]), "=&v"(rd[1]), "=&v"(rx[0]), "=&v"(rx[1])
                             : "v"(rows + d_row[0] * 4), "v"(rows + d_row[1] * 4), "v"(rows + x_row[0] * 4), "v"(rows + x_row[1] * 4) : "memory");
#pragma unroll
            for (int i = 0; i < ND; ++i)
                copy_piece(rd[i] >= 0 ? (const void*)((const T*)p.dy + rd[i] * p.dy_ld + d_col[i]) : (const void*)&ZERO_PIECE, to + (wave * ND + i) * 1024);
#pragma unroll
            for (int i = 0; i < NX; ++i)
                copy_piece(rx[i] >= 0 ? (const void*)((const T*)p.x + rx[i] * p.x_ld + x_col[i]) : (const void*)&ZERO_PIECE, to + D_BYTES + (wave * NX + i) * 1024);
            if (c_step + 1 < steps) ++c_step;                               // behind the last step the last one is copied again
            c_buf = c_buf == 2 ? 0 : c_buf + 1;
        };
        auto add_rows = [&](const typename El<T>::frag (&d)[MI], int u) {
            if (!bias || u != wk) return;
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int e = 0; e < E; ++e) sum[i] += (float)d[i][e];
        };
        auto end_step = [&](int s) {
            if ((s + 1) % PER_TILE) return;
            const int i = s / PER_TILE;
            const int g = __builtin_amdgcn_readfirstlane(lds_int(grp0 + i * 4)), next = __builtin_amdgcn_readfirstlane(lds_int(grp0 + i * 4 + 4));
            if (g != next) {
                settle<T, MI, NJ>(acc);
                flush(g);
                clear();
            }
        };
        wait_copies<0>();
        copy_step();
        copy_step();
        int buf = 0;
        typename El<T>::frag d[MI], x[NJ];
        copy_step();
        wait_copies<2 * COPIES>();
        __builtin_amdgcn_s_barrier();
#pragma unroll
        for (int i = 0; i < MI; ++i) d[i] = read_tr<T, BD * (int)sizeof(T)>(fd[0][i]);
#pragma unroll
        for (int j = 0; j < NJ; ++j) x[j] = read_tr<T, BX * (int)sizeof(T)>(fx[0][j]);
        for (int s = 0; s < steps; ++s) {
#pragma unroll
            for (int u = 0; u < S; ++u) {
                add_rows(d, u);
                if (u == S - 1) {
                    wait_copies<COPIES>();
                    __builtin_amdgcn_s_barrier();
                    buf = buf == 2 ? 0 : buf + 1;
                }
                const int n = (u + 1) % S;
                const unsigned stage = buf * STAGE;
                block_wgrad<BD * (int)sizeof(T), BX * (int)sizeof(T), NJ>(T(), acc, d, x, fd[n][0] + stage, fd[n][1] + stage, fx[n][0] + stage, fx[n][NJ - 1] + stage);
            }
            copy_step();
            end_step(s);
        }
        wait_copies<0>();                                                   // nothing may land once the rows are written anew
    }
}

// The same through registers, four waves per BT x BT block: any row length, any alignment (65 536 rows, 67 -> 256 bf16, 44 us).
template <typename T, int BT>
__global__ __launch_bounds__(THREADS, 2) void wgrad_kernel(WgradArgs p) {
    constexpr int E = piece<T>(), BK = step_len<T>();                       // rows of one step
    constexpr int PER_TILE = TILE_ROWS / BK, S = ROW_PIECES / 2;
    __shared__ __attribute__((aligned(16))) char lds[2 * tr_bytes<T, BT>()];
    __shared__ int tile_pos[MAX_CHUNK_TILES], tile_cnt[MAX_CHUNK_TILES], tile_grp[MAX_CHUNK_TILES];
    constexpr int M = BT / 64;                                              // 32 x 32 blocks of a wave: M x M
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n_off = (wave & 1) * (BT / 2), k_off = (wave >> 1) * (BT / 2);

    // the blocks of one chunk next to each other, on one XCD where there are eight chunks or more: they read the same rows
    const int G = p.rows.n_groups;
    const int tiles = grp::checked_tiles(p.rows.tile_base[G], p.rows.most_tiles);      // the rows of no group stay out
    const int blocks = p.tiles_n * p.tiles_k;
    const int64_t work = (int64_t)((tiles + p.chunk - 1) / p.chunk) * blocks;
    const int64_t per_xcd = (work + 7) / 8;
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
        const grp::Span span = grp::checked_span(p.rows.offsets[lo] + ((int64_t)t - p.rows.tile_base[lo]) * TILE_ROWS, p.rows.offsets[lo + 1], p.rows.n);
        tile_pos[i] = (int)span.pos;
        tile_cnt[i] = span.count;
        tile_grp[i] = lo;
    }
    __syncthreads();

    const int K = p.K, N = p.N;
    constexpr int BPR = BT / E, NP = BK * BPR / THREADS;                    // pieces of a row, of a thread
    char* const X = lds;
    char* const D = lds + tr_bytes<T, BT>();
    int prow[NP], pq[NP], rows[NP];
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        prow[j] = (tid + j * THREADS) / BPR;
        pq[j] = (tid + j * THREADS) % BPR;
    }
    Pack<T, E> rx[NP], rd[NP];
    const int steps = (t1 - t0) * PER_TILE;
    auto find = [&](int s) {                                                // rows of step s; -1 where it has none
        const int i = s < steps ? s / PER_TILE : 0, first = (s % PER_TILE) * BK;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int r = first + prow[j], cnt = tile_cnt[i];
            const int row = row_at(p.rows, (int64_t)tile_pos[i] + (r < cnt ? r : 0));
            rows[j] = s < steps && r < cnt ? row : -1;
        }
    };
    auto fill = [&]() {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const bool ok = rows[j] >= 0;
            const int64_t row = ok ? rows[j] : 0;
            const T *xrow = (const T*)p.x + row * p.x_ld, *drow = (const T*)p.dy + row * p.dy_ld;
            rx[j] = load_piece<T>(xrow, k0 + pq[j] * E, K, ok);
            rd[j] = load_piece<T>(drow, n0 + pq[j] * E, N, ok);
        }
    };
    f32x16 acc[M][M];
    float sum[M];                                                           // of dZ over this lane's rows
    auto clear = [&]() {
#pragma unroll
        for (int i = 0; i < M; ++i) {
            sum[i] = 0.0f;
#pragma unroll
            for (int j = 0; j < M; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
        }
    };
    const bool bias = p.db && k0 == 0 && k_off == 0;
    auto flush = [&](int g) {
        // within [0, tiles], so that a single chunk, which has no workspace, finishes every group
        const int b0 = grp::checked_tiles(p.rows.tile_base[g], tiles), b1 = grp::checked_tiles(p.rows.tile_base[g + 1], tiles);
        const bool whole = b0 >= t0 && b1 <= t1;
        const int64_t slot = 2 * (int64_t)c + (b0 >= t0 ? 1 : 0);
#pragma unroll
        for (int i = 0; i < M; ++i) {
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
            }
            if (bias) {
                const float s = sum[i] + __shfl_xor(sum[i], 32, 64);
                const int n = n0 + n_off + 32 * i + lane;
                if (lane < 32 && n < N) {
                    if (whole) ((T*)p.db)[(int64_t)g * N + n] = (T)s;
                    else p.part_b[slot * N + n] = s;
                }
            }
        }
    };

    clear();
    find(0);
    for (int s = 0; s < steps; ++s) {
        fill();                                                             // no registers left to hold a step ahead
        find(s + 1);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            put_piece<T, E>(X + tr_addr<T, BT>(prow[j], pq[j]), rx[j]);
            put_piece<T, E>(D + tr_addr<T, BT>(prow[j], pq[j]), rd[j]);
        }
        __syncthreads();
        typename El<T>::frag fx[S][M], fd[S][M];
#pragma unroll
        for (int u = 0; u < S; ++u)
#pragma unroll
            for (int i = 0; i < M; ++i) {
                fx[u][i] = tr_frag<T, BT>(X, k_off + 32 * i, u, lane);
                fd[u][i] = tr_frag<T, BT>(D, n_off + 32 * i, u, lane);
            }
        __syncthreads();                                                    // every wave has read the step
#pragma unroll
        for (int u = 0; u < S; ++u)
#pragma unroll
            for (int i = 0; i < M; ++i)
#pragma unroll
                for (int j = 0; j < M; ++j) acc[i][j] = El<T>::mfma(fd[u][i], fx[u][j], acc[i][j]);
        if (bias)
#pragma unroll
            for (int u = 0; u < S; ++u)
#pragma unroll
                for (int i = 0; i < M; ++i)
#pragma unroll
                    for (int e = 0; e < E; ++e) sum[i] += (float)fd[u][i][e];
        if ((s + 1) % PER_TILE == 0) {
            const int i = s / PER_TILE;
            if (i + 1 == t1 - t0 || tile_grp[i + 1] != tile_grp[i]) {
                flush(tile_grp[i]);
                clear();
            }
        }
    }
}

// Groups whose tiles lie in several chunks: the sum of their pieces in order; groups without rows: zeros.
template <typename T>
__global__ __launch_bounds__(THREADS) void wgrad_join_kernel(WgradArgs p, int64_t first) {
    const int g = blockIdx.y;
    const int b0 = grp::checked_tiles(p.rows.tile_base[g], p.rows.most_tiles), b1 = grp::checked_tiles(p.rows.tile_base[g + 1], p.rows.most_tiles);
    const unsigned chunk = (unsigned)p.chunk;                               // most workgroups end here: no signs to divide with
    const int c0 = (int)((unsigned)b0 / chunk), c1 = b1 > b0 ? (int)((unsigned)(b1 - 1) / chunk) : c0;
    if (b1 > b0 && c0 == c1) return;
    const int64_t NK = (int64_t)p.N * p.K;
    const int64_t i = first + (int64_t)blockIdx.x * THREADS + threadIdx.x;
    const bool is_w = i < NK;
    if (!is_w && !(p.db && i < NK + p.N)) return;
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

// Rows that are not whole pieces, copied to rows that are, for the streaming forms: with zeros behind the last column, or
// (SHIFT) the last piece ending where the row does, as out_of() has it.
template <typename T, bool SHIFT>
__global__ __launch_bounds__(THREADS) void pad_kernel(int64_t rows, int cols, const T* src, int64_t ld, T* dst) {
    constexpr int E = piece<T>();
    const int pieces = (cols + E - 1) / E;
    const int64_t total = rows * pieces;
    for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < total; i += (int64_t)gridDim.x * THREADS) {
        const int64_t row = total <= 0x7fffffff ? (int)i / pieces : i / pieces;
        const int c = (int)(i - row * pieces) * E;
        const T* from = src + row * ld;
        store_pack<T, E>(dst + i * E, SHIFT ? load_any<T, E>(from + min(c, cols - E)) : load_piece<T>(from, c, cols, true));
    }
}

// dZ = dY where the ReLU let something through.  Memory bound: 196 608 x 256 bf16 in 53 us, 5.7 TB/s; a layer of that size
// trains in 251 us with its ReLU and 190 without.  Written out once, because the gate inside the two products cost more when it
// was there: their tiles are bound by what they copy into LDS, and the gate is a third operand (data gradient 125 us gated and 59
// not, weight gradient 116 and 66, in short bursts of calls).
template <typename T>
__global__ __launch_bounds__(THREADS) void relu_bwd_kernel(int64_t n, int N, const T* dy, int64_t ld, const T* y, T* dz) {
    constexpr int E = piece<T>();
    const int pieces = (N + E - 1) / E;
    const int64_t total = n * pieces;
    for (int64_t i = (int64_t)blockIdx.x * THREADS + threadIdx.x; i < total; i += (int64_t)gridDim.x * THREADS) {
        const int64_t row = total <= 0x7fffffff ? (int)i / pieces : i / pieces;
        const int c = (int)(i - row * pieces) * E;
        Pack<T, E> g = load_piece<T>(dy + row * ld, c, N, true);
        gate_piece<T, E>(g, load_piece<T>(y + row * N, c, N, true));
        put_row_piece<T>(dz + row * N, c, N, g);
    }
}

static inline bool sizes_ok(int64_t n, int64_t n_groups, int K, int N) {
    return n >= 0 && n <= grp::MAX_ROWS && n_groups >= 1 && n_groups <= 65535 && K >= 1 && K <= 65536 && N >= 1 && N <= 65536;
}

// Operands whose rows are not whole pieces are copied to rows that are, and streamed, where that pays; a copy and its launch
// cost 5 us and up.  Measured, register form against copy and streaming form:
//   fp32, always from 2^28 products: 65 536 rows 63 -> 256 forward 80 / 47 us, data gradient 53 / 40, weight gradient 97 / 71
//   16 bits, forward: not (65 536 rows 67 -> 256 24 / 32, 196 608 rows 255 -> 257 126 / 150)
//   data gradient, weights alone: from 2^26 (4096 rows 67 -> 256 15 / 9.5, 65 536 rows 39 / 24); with dZ: from 2^31 (16 384 rows
//     250 -> 131 14 / 20, 65 536 rows 43 / 35, 196 608 rows 255 -> 257 155 / 120)
//   weight gradient, one operand: from 2^26 (65 536 rows 67 -> 256 44 / 30); both: from 2^31 (16 384 rows 250 -> 131 30 / 36,
//     65 536 rows 55 / 53, 196 608 rows 255 -> 257 302 / 183); not up to 64 x 64 (65 536 rows 63 -> 64 20 / 26)
struct PadPlan {
    bool fwd, data, weights;
    int Kp, Np;                                                             // whole pieces
};
static PadPlan pad_plan(int64_t n, int64_t n_groups, int K, int N, int precision) {
    const int E = 16 / elem_bytes(precision);
    PadPlan p = {};
    p.Kp = (K + E - 1) / E * E;
    p.Np = (N + E - 1) / E * E;
    const bool odd_k = K % E != 0, odd_n = N % E != 0, fp32 = precision == NERF_PREC_FP32;
    if (K < E || N < E || (K <= 64 && N <= 64) || n_groups * K * N > 4 * n * (K + N)) return p;
    const double products = (double)n * K * N;                              // n K N may pass 64 bits
    const double one = fp32 ? 0x1p28 : 0x1p26, two = fp32 ? 0x1p28 : 0x1p31;
    p.fwd = odd_k && fp32 && products >= one;
    p.data = (odd_k || odd_n) && products >= (odd_n ? two : one);
    p.weights = (odd_k || odd_n) && products >= (odd_k && odd_n ? two : one);
    return p;
}
static inline int64_t elems256(int64_t elems, int precision) { return (elems * elem_bytes(precision) + 255) / 256 * 256; }

static int pad_rows(int64_t rows, int cols, const void* src, int64_t ld, void* dst, bool shift, int precision, void* stream) {
    const int E = 16 / elem_bytes(precision);
    const int64_t blocks = (rows * ((cols + E - 1) / E) + THREADS - 1) / THREADS, most = (int64_t)1 << 22;
    const dim3 grid((unsigned)(blocks < most ? blocks : most));
#define NERF_CALL(T)                                                                                                                       \
    do {                                                                                                                                   \
        if (shift) hipLaunchKernelGGL((pad_kernel<T, true>), grid, dim3(THREADS), 0, (hipStream_t)stream, rows, cols, (const T*)src, ld, (T*)dst); \
        else hipLaunchKernelGGL((pad_kernel<T, false>), grid, dim3(THREADS), 0, (hipStream_t)stream, rows, cols, (const T*)src, ld, (T*)dst);      \
    } while (0)
    NERF_ELEM_DISPATCH(precision, NERF_CALL);
#undef NERF_CALL
    return nerf_launch_status();
}

// workgroups of a grid whose kernel gives each of the eight XCDs an equal run of `work`
static inline int64_t xcd_grid(int64_t work) { return (work + 7) / 8 * 8; }

struct WgradPlan {
    int bd, bx, tiles_n, tiles_k, chunk;
    int64_t chunks, part_w, part_b, bytes;
};
// wide: whole aligned pieces (one workgroup per compute unit), else through registers (two)
static WgradPlan wgrad_plan(int64_t n, int64_t n_groups, int K, int N, bool wide, int precision) {
    WgradPlan w = {};
    w.bd = !wide && K <= 64 && N <= 64 ? 64 : 128;
    w.bx = wide && precision != NERF_PREC_FP32 && K > 128 ? 256 : w.bd;
    w.tiles_n = (N + w.bd - 1) / w.bd;
    w.tiles_k = (K + w.bx - 1) / w.bx;
    const int64_t tiles = grp::max_tiles(n, n_groups), blocks = (int64_t)w.tiles_n * w.tiles_k;
    int64_t chunks = (wide ? 256 : 512) / blocks;
    if (chunks < 1) chunks = 1;
    int64_t chunk = (tiles + chunks - 1) / chunks;
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
    hipStream_t st = (hipStream_t)stream;
    const int64_t tiles = grp::max_tiles(p.rows.n, p.rows.n_groups);
    if (wide) {
        // Output tile: the width with the least work on the busiest compute unit, ceil(items / 256) tiles of BN + an
        // overhead for reading the rows once more per tile (which weighs more where the products are fast).
        const int most = precision == NERF_PREC_FP32 ? 128 : 256, extra = precision == NERF_PREC_FP32 ? 8 : 32;
        int bn = 64;
        int64_t least = -1;
        for (int b = 64; b <= most; b *= 2) {
            const int64_t cost = (tiles * ((p.O + b - 1) / b) + 255) / 256 * (b + extra);
            if (least < 0 || cost < least) { least = cost; bn = b; }
        }
        p.tiles_o = (p.O + bn - 1) / bn;
        int64_t grid = (tiles * p.tiles_o + 7) / 8 * 8;
        if (grid > (bn == 64 ? 512 : 256)) grid = bn == 64 ? 512 : 256;
#define NERF_ST(T, BN) hipLaunchKernelGGL((stream_kernel<T, WT, BN>), dim3((unsigned)grid), dim3(ST_THREADS), 0, st, p)
#define NERF_CALL(T)                                                \
    do {                                                            \
        if constexpr (sizeof(T) == 2)                               \
            if (bn == 256) { NERF_ST(T, 256); break; }              \
        if (bn == 128) NERF_ST(T, 128);                             \
        else NERF_ST(T, 64);                                        \
    } while (0)
        NERF_ELEM_DISPATCH(precision, NERF_CALL);
#undef NERF_CALL
#undef NERF_ST
        return nerf_launch_status();
    }
    const int bn = p.O <= 64 ? 64 : 128;
    p.tiles_o = (p.O + bn - 1) / bn;
    // many groups times many outputs: more workgroups than a direction of the grid holds threads for go to the next one
    const int64_t work = xcd_grid(tiles * p.tiles_o), row = work < MAX_GRID ? work : MAX_GRID;
    NERF_REQUIRE((work + row - 1) / row < 65536, NERF_E_SHAPE);
    const dim3 grid((unsigned)row, (unsigned)((work + row - 1) / row));
    p.grid_row = (int)(row / 8);
#define NERF_CALL(T)                                                                                                           \
    do {                                                                                                                       \
        if (bn == 128) hipLaunchKernelGGL((linear_kernel<T, WT, 128>), grid, dim3(THREADS), 0, st, p);                         \
        else hipLaunchKernelGGL((linear_kernel<T, WT, 64>), grid, dim3(THREADS), 0, st, p);                                    \
    } while (0)
    NERF_ELEM_DISPATCH(precision, NERF_CALL);
#undef NERF_CALL
    return nerf_launch_status();
}

}  // namespace gl
}  // namespace nerf

extern "C" int64_t nerf_grouped_workspace_bytes(int64_t n, int64_t n_groups, int K, int N, int backward, int precision) {
    using namespace nerf;
    if (!gl::sizes_ok(n, n_groups, K, N)) return NERF_E_SHAPE;
    if (!elem_ok(precision)) return NERF_E_DTYPE;
    const gl::PadPlan p = gl::pad_plan(n, n_groups, K, N, precision);
    if (!(backward ? p.data : p.fwd)) return 0;
    return gl::elems256(n * (backward ? p.Np : p.Kp), precision) + gl::elems256(n_groups * N * p.Kp, precision);
}

extern "C" int nerf_grouped_fwd(int64_t n, int64_t n_groups, const int32_t* order, const int32_t* offsets, const int32_t* tile_base,
                                int K, int N, const void* x, int64_t x_ld, const void* weight, const void* bias, int relu,
                                int precision, void* y, void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace nerf;
    NERF_REQUIRE(gl::sizes_ok(n, n_groups, K, N) && x_ld >= K, NERF_E_SHAPE);
    NERF_REQUIRE(elem_ok(precision), NERF_E_DTYPE);
    if (n == 0) return NERF_OK;
    const gl::PadPlan pad = gl::pad_plan(n, n_groups, K, N, precision);
    NERF_REQUIRE(order && offsets && tile_base && x && weight && y && (workspace || !pad.fwd), NERF_E_NULL);
    const int es = elem_bytes(precision), E = 16 / es;
    NERF_REQUIRE(nerf_aligned(x, (uintptr_t)es) && nerf_aligned(weight, (uintptr_t)es) && nerf_aligned(y, (uintptr_t)es) &&
                 nerf_aligned(bias, (uintptr_t)es) && nerf_aligned(workspace, 256), NERF_E_ALIGN);
    NERF_REQUIRE(workspace_bytes >= nerf_grouped_workspace_bytes(n, n_groups, K, N, 0, precision), NERF_E_WORKSPACE);
    gl::LinArgs p = {};
    p.rows = {n, (int)n_groups, (int)grp::max_tiles(n, n_groups), order, offsets, tile_base};
    p.C = K; p.O = N; p.a = x; p.a_ld = x_ld; p.w = weight; p.w_ld = K; p.w_gs = (int64_t)N * K; p.bias = bias; p.relu = relu ? 1 : 0; p.out = y;
    const bool whole = K % E == 0 && x_ld % E == 0 && nerf_aligned(x, 16) && nerf_aligned(weight, 16) && N >= E;
    if (pad.fwd) {
        void *a = workspace, *w = (char*)workspace + gl::elems256(n * pad.Kp, precision);
        int rc = gl::pad_rows(n, K, x, x_ld, a, false, precision, stream);
        if (rc == NERF_OK) rc = gl::pad_rows(n_groups * N, K, weight, K, w, false, precision, stream);
        if (rc != NERF_OK) return rc;
        p.C = pad.Kp; p.a = a; p.a_ld = pad.Kp; p.w = w; p.w_ld = pad.Kp; p.w_gs = (int64_t)N * pad.Kp;
        return gl::launch_linear<false>(p, precision, true, stream);
    }
    return gl::launch_linear<false>(p, precision, whole, stream);
}

extern "C" int nerf_relu_bwd(int64_t n, int N, const void* d_y, int64_t d_y_ld, const void* y, int precision, void* d_z, void* stream) {
    using namespace nerf;
    NERF_REQUIRE(gl::sizes_ok(n, 1, 1, N) && d_y_ld >= N, NERF_E_SHAPE);
    NERF_REQUIRE(elem_ok(precision), NERF_E_DTYPE);
    if (n == 0) return NERF_OK;
    NERF_REQUIRE(d_y && y && d_z, NERF_E_NULL);
    const int es = elem_bytes(precision), E = 16 / es;
    NERF_REQUIRE(nerf_aligned(d_y, (uintptr_t)es) && nerf_aligned(y, (uintptr_t)es) && nerf_aligned(d_z, (uintptr_t)es), NERF_E_ALIGN);
    const int64_t pieces = n * ((N + E - 1) / E), most = (int64_t)1 << 22;
    const unsigned grid = (unsigned)((pieces + gl::THREADS - 1) / gl::THREADS < most ? (pieces + gl::THREADS - 1) / gl::THREADS : most);
#define NERF_CALL(T) \
    hipLaunchKernelGGL(gl::relu_bwd_kernel<T>, dim3(grid), dim3(gl::THREADS), 0, (hipStream_t)stream, n, N, (const T*)d_y, d_y_ld, (const T*)y, (T*)d_z)
    NERF_ELEM_DISPATCH(precision, NERF_CALL);
#undef NERF_CALL
    return nerf_launch_status();
}

extern "C" int nerf_grouped_bwd_data(int64_t n, int64_t n_groups, const int32_t* order, const int32_t* offsets, const int32_t* tile_base,
                                     int K, int N, const void* d_z, int64_t d_z_ld, const void* weight, int precision, void* d_x,
                                     void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace nerf;
    NERF_REQUIRE(gl::sizes_ok(n, n_groups, K, N) && d_z_ld >= N, NERF_E_SHAPE);
    NERF_REQUIRE(elem_ok(precision), NERF_E_DTYPE);
    if (n == 0) return NERF_OK;
    const gl::PadPlan pad = gl::pad_plan(n, n_groups, K, N, precision);
    NERF_REQUIRE(order && offsets && tile_base && d_z && weight && d_x && (workspace || !pad.data), NERF_E_NULL);
    const int es = elem_bytes(precision), E = 16 / es;
    NERF_REQUIRE(nerf_aligned(d_z, (uintptr_t)es) && nerf_aligned(weight, (uintptr_t)es) && nerf_aligned(d_x, (uintptr_t)es) &&
                 nerf_aligned(workspace, 256), NERF_E_ALIGN);
    NERF_REQUIRE(workspace_bytes >= nerf_grouped_workspace_bytes(n, n_groups, K, N, 1, precision), NERF_E_WORKSPACE);
    gl::LinArgs p = {};
    p.rows = {n, (int)n_groups, (int)grp::max_tiles(n, n_groups), order, offsets, tile_base};
    p.C = N; p.O = K; p.a = d_z; p.a_ld = d_z_ld; p.w = weight; p.w_ld = K; p.w_gs = (int64_t)N * K; p.w_rows = N; p.out = d_x;
    bool a_whole = N % E == 0 && d_z_ld % E == 0 && nerf_aligned(d_z, 16), w_whole = K % E == 0 && nerf_aligned(weight, 16);
    if (pad.data && (a_whole || N % E) && (w_whole || K % E)) {
        if (!a_whole) {
            const int rc = gl::pad_rows(n, N, d_z, d_z_ld, workspace, false, precision, stream);
            if (rc != NERF_OK) return rc;
            p.C = pad.Np; p.a = workspace; p.a_ld = pad.Np;
        }
        if (!w_whole) {
            void* w = (char*)workspace + gl::elems256(n * pad.Np, precision);
            const int rc = gl::pad_rows(n_groups * N, K, weight, K, w, true, precision, stream);
            if (rc != NERF_OK) return rc;
            p.w = w; p.w_ld = pad.Kp; p.w_gs = (int64_t)N * pad.Kp;
        }
        a_whole = w_whole = true;
    }
    return gl::launch_linear<true>(p, precision, a_whole && w_whole, stream);
}

namespace nerf {
namespace gl {
// for the pieces of dW: alignment decides the form, and with it the number of chunks; enough for either
static int64_t wgrad_bytes(int64_t n, int64_t n_groups, int K, int N, int precision) {
    const int64_t a = wgrad_plan(n, n_groups, K, N, false, precision).bytes, b = wgrad_plan(n, n_groups, K, N, true, precision).bytes;
    return ((a > b ? a : b) + 255) / 256 * 256;
}
}  // namespace gl
}  // namespace nerf

extern "C" int64_t nerf_grouped_bwd_weights_workspace_bytes(int64_t n, int64_t n_groups, int K, int N, int precision) {
    using namespace nerf;
    if (!gl::sizes_ok(n, n_groups, K, N)) return NERF_E_SHAPE;
    if (!elem_ok(precision)) return NERF_E_DTYPE;
    const gl::PadPlan pad = gl::pad_plan(n, n_groups, K, N, precision);
    return gl::wgrad_bytes(n, n_groups, K, N, precision) + (pad.weights ? gl::elems256(n * pad.Kp, precision) + gl::elems256(n * pad.Np, precision) : 0);
}

extern "C" int nerf_grouped_bwd_weights(int64_t n, int64_t n_groups, const int32_t* order, const int32_t* offsets,
                                        const int32_t* tile_base, int K, int N, const void* d_z, int64_t d_z_ld, const void* x,
                                        int64_t x_ld, int precision, void* d_weight, void* d_bias, void* workspace,
                                        int64_t workspace_bytes, void* stream) {
    using namespace nerf;
    NERF_REQUIRE(gl::sizes_ok(n, n_groups, K, N) && d_z_ld >= N && x_ld >= K, NERF_E_SHAPE);
    NERF_REQUIRE(elem_ok(precision), NERF_E_DTYPE);
    if (n == 0) return NERF_OK;
    NERF_REQUIRE(order && offsets && tile_base && d_z && x && d_weight && workspace, NERF_E_NULL);
    const int es = elem_bytes(precision), E = 16 / es;
    NERF_REQUIRE(nerf_aligned(d_z, (uintptr_t)es) && nerf_aligned(x, (uintptr_t)es) && nerf_aligned(d_weight, (uintptr_t)es) &&
                 nerf_aligned(d_bias, (uintptr_t)es) && nerf_aligned(workspace, 256), NERF_E_ALIGN);
    NERF_REQUIRE(workspace_bytes >= nerf_grouped_bwd_weights_workspace_bytes(n, n_groups, K, N, precision), NERF_E_WORKSPACE);
    // Up to 64 x 64 the register form has blocks of that size, a quarter of the streaming form's products: 64 -> 64 fp32 53 us
    // against 89 (196 608 rows) and 12.5 against 19.5 (1024); bf16 12.5 against 16 at 16 384 rows, but 31 against 26.5 at 196 608.
    const bool small = K <= 64 && N <= 64 && (precision == NERF_PREC_FP32 || n < 65536);
    const gl::PadPlan pad = gl::pad_plan(n, n_groups, K, N, precision);
    bool d_whole = N % E == 0 && d_z_ld % E == 0 && nerf_aligned(d_z, 16), x_whole = K % E == 0 && x_ld % E == 0 && nerf_aligned(x, 16);
    if (pad.weights && (d_whole || N % E) && (x_whole || K % E)) {
        char* at = (char*)workspace + gl::wgrad_bytes(n, n_groups, K, N, precision);
        if (!x_whole) {
            const int rc = gl::pad_rows(n, K, x, x_ld, at, false, precision, stream);
            if (rc != NERF_OK) return rc;
            x = at; x_ld = pad.Kp;
        }
        if (!d_whole) {
            at += gl::elems256(n * pad.Kp, precision);
            const int rc = gl::pad_rows(n, N, d_z, d_z_ld, at, false, precision, stream);
            if (rc != NERF_OK) return rc;
            d_z = at; d_z_ld = pad.Np;
        }
        d_whole = x_whole = true;
    }
    const bool wide = !small && d_whole && x_whole;
    const gl::WgradPlan w = gl::wgrad_plan(n, n_groups, K, N, wide, precision);
    gl::WgradArgs p = {};
    p.rows = {n, (int)n_groups, (int)grp::max_tiles(n, n_groups), order, offsets, tile_base};
    p.K = K; p.N = N; p.Kp = pad.Kp; p.Np = pad.Np; p.tiles_k = w.tiles_k; p.tiles_n = w.tiles_n; p.chunk = w.chunk;
    p.x_ld = x_ld; p.dy_ld = d_z_ld; p.x = x; p.dy = d_z; p.dw = d_weight; p.db = d_bias;
    p.part_w = (float*)((char*)workspace + w.part_w);
    p.part_b = (float*)((char*)workspace + w.part_b);
    const int64_t blocks = (int64_t)w.tiles_n * w.tiles_k;
    const int64_t grid = gl::xcd_grid(w.chunks * blocks);
    NERF_REQUIRE(grid <= 2 * gl::MAX_GRID - 8, NERF_E_SHAPE);               // 512 threads each
    hipStream_t st = (hipStream_t)stream;
    const int64_t join_blocks = ((int64_t)N * K + N + gl::THREADS - 1) / gl::THREADS;
#define NERF_WG(T, BT) hipLaunchKernelGGL((gl::wgrad_kernel<T, BT>), dim3((unsigned)grid), dim3(gl::THREADS), 0, st, p)
#define NERF_WS(T, BX) hipLaunchKernelGGL((gl::wgrad_stream_kernel<T, BX>), dim3((unsigned)grid), dim3(gl::ST_THREADS), 0, st, p)
#define NERF_CALL(T)                                                                                   \
    do {                                                                                               \
        bool done = false;                                                                             \
        if constexpr (sizeof(T) == 2)                                                                  \
            if (w.bx == 256) { NERF_WS(T, 256); done = true; }                                         \
        if (done) {}                                                                                   \
        else if (wide) NERF_WS(T, 128);                                                                \
        else if (w.bd == 128) NERF_WG(T, 128);                                                         \
        else NERF_WG(T, 64);                                                                           \
        for (int64_t b = 0; b < join_blocks; b += gl::MAX_GRID) {                                      \
            const dim3 join((unsigned)(join_blocks - b < gl::MAX_GRID ? join_blocks - b : gl::MAX_GRID), (unsigned)n_groups); \
            hipLaunchKernelGGL(gl::wgrad_join_kernel<T>, join, dim3(gl::THREADS), 0, st, p, b * gl::THREADS); \
        }                                                                                              \
    } while (0)
    NERF_ELEM_DISPATCH(precision, NERF_CALL);
#undef NERF_CALL
#undef NERF_WS
#undef NERF_WG
    return nerf_launch_status();
}
