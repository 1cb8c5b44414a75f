// Grouping of rows by an integer id: the stable order that puts the rows of one group next to each other, where each
// group begins, and how many 128-row tiles the groups before it hold.  The reference has no sub-networks; this is what
// hands sample points to them (nerf_grouped_fwd) and what the gradient of a row look-up sums by (nerf_embed_bwd).
//
// An LSD radix sort of (id, position); ids outside [0, n_groups) take the key n_groups and come last.  For a digit every
// wave owns a run of consecutive positions.  The lanes of one 64-element round that hold the same digit find each other
// with one ballot per bit, so equal digits keep their order and a digit's count is one LDS addition however many lanes
// hold it (the samples of a ray share an id).  An exclusive sum over (digit, wave) gives each wave its first place per
// digit.  Only integers are added, so the result does not depend on timing.
//
// Up to SMALL_N rows one workgroup keeps everything in LDS (one launch, digits of at most 8 bits).  Above, three launches
// per digit of at most 11 bits: counts per block of rows, an exclusive sum per digit over the blocks, and the ranked
// scatter.  A wide digit costs more counters per block (8 KiB per wave at 11 bits) but saves a whole pass: ids of 256 to
// 2047 groups take one, of up to four million two.
#include "groups.hpp"

namespace nerf {
namespace grp {

constexpr int SMALL_N = 2048;      // rows one workgroup sorts in LDS: 1024 rows take 6 us, 4096 would take 14, as many as 200 000 in blocks
constexpr int SMALL_THREADS = 1024;
constexpr int BLOCK_THREADS = 256;
constexpr int MAX_BITS = 11;        // of a digit above SMALL_N rows
constexpr int SCAN_DIGITS = 16;     // digits of a workgroup of the sum over the blocks: one per wave

template <typename ID>
__device__ __forceinline__ unsigned key_of(const ID* ids, int64_t i, unsigned n_groups) {
    const ID v = ids[i];
    return v >= 0 && v < (ID)n_groups ? (unsigned)v : n_groups;
}

// the lanes of the wave (out of `active`) that hold the same digit as this one
__device__ __forceinline__ unsigned long long same_digit(unsigned digit, int bits, unsigned long long active) {
    unsigned long long m = active;
    for (int b = 0; b < bits; ++b) {
        const unsigned long long s = __ballot((digit >> b) & 1u);
        m &= (digit >> b) & 1u ? s : ~s;
    }
    return m;
}

__device__ __forceinline__ int wave_incl_add(int v, int lane) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int u = __shfl_up(v, off, 64);
        if (lane >= off) v += u;
    }
    return v;
}

// exclusive sum over the threads of a block of WAVES waves; `total` = sum over all.  part: WAVES ints of LDS.
template <int WAVES>
__device__ __forceinline__ int block_excl_add(int v, int* part, int* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int incl = wave_incl_add(v, lane);
    if (lane == 63) part[wave] = incl;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const int t = part[w];
        if (w < wave) before += t;
        all += t;
    }
    __syncthreads();
    *total = all;
    return before + incl - v;
}

// tile_base from the group boundaries: `begin(g)` for g in [0, n_groups], the rows behind the last group count as one
// more group.  All threads of the block take part.
template <int WAVES, typename F>
__device__ __forceinline__ void write_tile_base(F begin, int n, int n_groups, int* part, int32_t* tile_base) {
    int carry = 0;
    for (int g0 = 0; g0 <= n_groups; g0 += WAVES * 64) {
        const int g = g0 + (int)threadIdx.x;
        int tiles = 0;
        if (g <= n_groups) {
            const int lo = begin(g), hi = g < n_groups ? begin(g + 1) : n;
            tiles = (hi - lo) / TILE_ROWS + ((hi - lo) % TILE_ROWS != 0);
        }
        int all;
        const int excl = block_excl_add<WAVES>(tiles, part, &all);
        if (g <= n_groups) {
            tile_base[g] = carry + excl;
            if (g == n_groups) tile_base[g + 1] = carry + excl + tiles;
        }
        carry += all;
    }
}

// n <= SMALL_N: the whole sort in one workgroup.  `passes` digits of `bits` bits.  offsets / tile_base are written
// here when there is one digit; with more, offsets_kernel follows (it needs the sorted keys).
template <typename ID>
__global__ __launch_bounds__(SMALL_THREADS) void small_kernel(int n, const ID* __restrict__ ids, int n_groups, int passes,
                                                              int bits, int32_t* __restrict__ order, int32_t* __restrict__ offsets,
                                                              int32_t* __restrict__ tile_base, int32_t* __restrict__ keys) {
    __shared__ unsigned lk[SMALL_N];
    __shared__ unsigned short li[SMALL_N];
    __shared__ int cnt[SMALL_THREADS / 64][256];
    __shared__ int offs[257];
    __shared__ int part[SMALL_THREADS / 64];
    constexpr int ROUNDS = SMALL_N / SMALL_THREADS;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // the rows in front of n are dealt out to the waves in equal runs of whole rounds
    const int per_wave = ((n + SMALL_THREADS - 1) / SMALL_THREADS) * 64;
    unsigned k[ROUNDS];
    unsigned short at[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int p = wave * per_wave + r * 64 + lane;
        const bool ok = r * 64 < per_wave && p < n;
        k[r] = ok ? key_of(ids, p, (unsigned)n_groups) : 0u;
        at[r] = (unsigned short)p;
    }
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * bits;
        const unsigned mask = (1u << bits) - 1u;
        for (int i = tid; i < SMALL_THREADS / 64 * 256; i += SMALL_THREADS) (&cnt[0][0])[i] = 0;
        __syncthreads();
        if (pass > 0) {
#pragma unroll
            for (int r = 0; r < ROUNDS; ++r) {
                const int p = wave * per_wave + r * 64 + lane;
                if (r * 64 < per_wave && p < n) { k[r] = lk[p]; at[r] = li[p]; }
            }
        }
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const int p = wave * per_wave + r * 64 + lane;
            if (r * 64 < per_wave && p < n) atomicAdd(&cnt[wave][(k[r] >> shift) & mask], 1);
        }
        __syncthreads();
        // thread t: digit t / 4, waves 4 (t % 4) .. + 3
        const int d = tid >> 2, w0 = (tid & 3) * 4;
        int c[4], sum = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) { c[j] = cnt[w0 + j][d]; sum += c[j]; }
        int all;
        int run = block_excl_add<SMALL_THREADS / 64>(sum, part, &all);
        if ((tid & 3) == 0) offs[d] = run;
#pragma unroll
        for (int j = 0; j < 4; ++j) { cnt[w0 + j][d] = run; run += c[j]; }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const int p = wave * per_wave + r * 64 + lane;
            const bool ok = r * 64 < per_wave && p < n;
            const unsigned dig = (k[r] >> shift) & mask;
            const unsigned long long peers = same_digit(dig, bits, __ballot(ok));
            if (ok) {
                const int rank = __popcll(peers & ((1ull << lane) - 1ull));
                const int to = cnt[wave][dig] + rank;
                lk[to] = k[r];
                li[to] = at[r];
            }
            wave_lds_sync();                                     // every lane has read its place before it moves on
            if (ok && (peers >> lane) == 1ull) cnt[wave][dig] += __popcll(peers);   // the last lane of each digit
            wave_lds_sync();
        }
        __syncthreads();
    }
    for (int p = tid; p < n; p += SMALL_THREADS) {
        order[p] = li[p];
        if (keys) keys[p] = (int32_t)lk[p];
    }
    if (passes == 1) {
        for (int g = tid; g <= n_groups; g += SMALL_THREADS) offsets[g] = offs[g];
        if (tile_base) write_tile_base<SMALL_THREADS / 64>([&](int g) { return offs[g]; }, n, n_groups, part, tile_base);
    }
}

// digit counts of each block of ROUNDS * BLOCK_THREADS rows: hist[block][digit]
template <typename ID, int ROUNDS>
__global__ __launch_bounds__(BLOCK_THREADS) void hist_kernel(int64_t n, const ID* __restrict__ ids, unsigned n_groups, int shift,
                                                             int bits, int32_t* __restrict__ hist) {
    extern __shared__ int cnt[];                                   // [1 << bits]
    const int tid = threadIdx.x, lane = tid & 63, bins = 1 << bits;
    const int64_t p0 = (int64_t)blockIdx.x * (ROUNDS * BLOCK_THREADS) + tid;
    unsigned k[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int64_t p = p0 + r * BLOCK_THREADS;
        k[r] = p < n ? (key_of(ids, p, n_groups) >> shift) & (unsigned)(bins - 1) : 0u;
    }
    for (int d = tid; d < bins; d += BLOCK_THREADS) cnt[d] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const bool ok = p0 + r * BLOCK_THREADS < n;
        const unsigned long long peers = same_digit(k[r], bits, __ballot(ok));
        if (ok && (peers >> lane) == 1ull) atomicAdd(&cnt[k[r]], __popcll(peers));
    }
    __syncthreads();
    for (int d = tid; d < bins; d += BLOCK_THREADS) hist[(int64_t)blockIdx.x * bins + d] = cnt[d];
}

// Exclusive sum of each digit's counts over the blocks, in place, and the digit's total.  A workgroup owns 16 digits (64
// bytes of a block's counts) and takes 512 blocks at a time: thread (digit, chunk) keeps the counts of 8 blocks in registers,
// a wave adds up one digit's 64 chunks.  With the counts of a block side by side, blocks write and read them in whole lines
// (digit by digit, 524 288 ids over 65 536 rows took 52 us, now 48).
__global__ __launch_bounds__(SCAN_DIGITS * 64) void colscan_kernel(int nblk, int bins, int32_t* __restrict__ hist, int32_t* __restrict__ totals) {
    constexpr int PER = 8;
    __shared__ int part[64][SCAN_DIGITS + 1], whole[SCAN_DIGITS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, dl = tid % SCAN_DIGITS, chunk = tid / SCAN_DIGITS;
    const int d = (int)blockIdx.x * SCAN_DIGITS + dl;
    int carry = 0;
    for (int64_t b0 = 0; b0 < nblk; b0 += 64 * PER) {
        int v[PER], sum = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int64_t b = b0 + chunk * PER + j;
            v[j] = d < bins && b < nblk ? hist[b * bins + d] : 0;
            sum += v[j];
        }
        part[chunk][dl] = sum;
        __syncthreads();
        const int x = part[lane][wave];
        int incl = x;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int u = __shfl_up(incl, off, 64);
            if (lane >= off) incl += u;
        }
        part[lane][wave] = incl - x;
        if (lane == 63) whole[wave] = incl;
        __syncthreads();
        int run = carry + part[chunk][dl];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int64_t b = b0 + chunk * PER + j;
            if (d < bins && b < nblk) hist[b * bins + d] = run;
            run += v[j];
        }
        carry += whole[dl];
        __syncthreads();
    }
    if (chunk == 0 && d < bins) totals[d] = carry;
}

// ranked scatter of one digit.  idx_in: the positions that belong to the keys (NULL in the first pass: the row itself).
// offsets / tile_base are written by block 0 when `single` (the digit is the whole key).
template <typename ID, int ROUNDS>
__global__ __launch_bounds__(BLOCK_THREADS) void scatter_kernel(int64_t n, const ID* __restrict__ ids, const int32_t* __restrict__ idx_in,
                                                                unsigned n_groups, int shift, int bits,
                                                                const int32_t* __restrict__ hist, const int32_t* __restrict__ totals,
                                                                int32_t* __restrict__ key_out, int32_t* __restrict__ idx_out, int single,
                                                                int32_t* __restrict__ offsets, int32_t* __restrict__ tile_base) {
    constexpr int WAVES = BLOCK_THREADS / 64;
    constexpr int PER = (1 << MAX_BITS) / BLOCK_THREADS;           // digits of a thread in the exclusive sum, at most
    extern __shared__ int cnt[];                                   // [WAVES][1 << bits], then [1 << bits] first places
    __shared__ int part[WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, bins = 1 << bits;
    int* mine = cnt + wave * bins;
    int* offs = cnt + WAVES * bins;
    const int64_t p0 = (int64_t)blockIdx.x * (ROUNDS * BLOCK_THREADS) + wave * (ROUNDS * 64) + lane;
    unsigned k[ROUNDS];
    int at[ROUNDS];
    unsigned long long peers[ROUNDS];
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const int64_t p = p0 + r * 64;
        k[r] = p < n ? key_of(ids, p, n_groups) : 0u;
        at[r] = p < n ? (idx_in ? idx_in[p] : (int)p) : 0;
    }
    const int per = bins > BLOCK_THREADS ? bins / BLOCK_THREADS : 1;
    int total[PER], before[PER], sum = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int d = tid * per + j;
        const bool on = j < per && d < bins;
        total[j] = on ? totals[d] : 0;
        before[j] = on ? hist[(int64_t)blockIdx.x * bins + d] : 0;
        sum += total[j];
    }
    for (int i = tid; i < WAVES * bins; i += BLOCK_THREADS) cnt[i] = 0;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const bool ok = p0 + r * 64 < n;
        const unsigned dig = (k[r] >> shift) & (unsigned)(bins - 1);
        peers[r] = same_digit(dig, bits, __ballot(ok));
        if (ok && (peers[r] >> lane) == 1ull) atomicAdd(&mine[dig], __popcll(peers[r]));
    }
    int all;
    int first = block_excl_add<WAVES>(sum, part, &all);            // (its barriers also publish the counts)
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int d = tid * per + j;
        if (j >= per || d >= bins) continue;
        offs[d] = first;
        int run = first + before[j];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) { const int c = cnt[w * bins + d]; cnt[w * bins + d] = run; run += c; }
        first += total[j];
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) {
        const bool ok = p0 + r * 64 < n;
        const unsigned dig = (k[r] >> shift) & (unsigned)(bins - 1);
        if (ok) {
            const int to = mine[dig] + __popcll(peers[r] & ((1ull << lane) - 1ull));
            idx_out[to] = at[r];
            if (key_out) key_out[to] = (int32_t)k[r];
        }
        wave_lds_sync();
        if (ok && (peers[r] >> lane) == 1ull) mine[dig] += __popcll(peers[r]);
        wave_lds_sync();
    }
    if (single && blockIdx.x == 0) {
        for (int g = tid; g <= (int)n_groups; g += BLOCK_THREADS) offsets[g] = offs[g];
        if (tile_base)
            write_tile_base<WAVES>([&](int g) { return offs[g]; }, (int)n, (int)n_groups, part, tile_base);
    }
}

// offsets[g] = number of sorted keys below g
__global__ __launch_bounds__(BLOCK_THREADS) void offsets_kernel(int64_t n, const int32_t* __restrict__ keys, int n_groups,
                                                                int32_t* __restrict__ offsets) {
    const int64_t g = (int64_t)blockIdx.x * BLOCK_THREADS + threadIdx.x;
    if (g > n_groups) return;
    int64_t lo = 0, hi = n;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if (keys[mid] < (int32_t)g) lo = mid + 1;
        else hi = mid;
    }
    offsets[g] = (int32_t)lo;
}

__global__ __launch_bounds__(SMALL_THREADS) void tile_base_kernel(int n, int n_groups, const int32_t* __restrict__ offsets,
                                                                  int32_t* __restrict__ tile_base) {
    __shared__ int part[SMALL_THREADS / 64];
    write_tile_base<SMALL_THREADS / 64>([&](int g) { return offsets[g]; }, n, n_groups, part, tile_base);
}

// The caller's own boundaries made safe to index with: 0 first, never below the one before, never above n.
__global__ __launch_bounds__(SMALL_THREADS) void clean_offsets_kernel(int n, int n_groups, const int32_t* __restrict__ in,
                                                                      int32_t* __restrict__ offsets) {
    __shared__ int part[SMALL_THREADS / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int carry = 0;
    for (int g0 = 0; g0 <= n_groups; g0 += SMALL_THREADS) {
        const int g = g0 + (int)threadIdx.x;
        int v = g == 0 || g > n_groups ? 0 : min(max(in[g], 0), n);
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int u = __shfl_up(v, off, 64);
            if (lane >= off) v = max(v, u);
        }
        if (lane == 63) part[wave] = v;
        __syncthreads();
        int top = carry;
        for (int w = 0; w < SMALL_THREADS / 64; ++w) {
            if (w < wave) v = max(v, part[w]);
            top = max(top, part[w]);
        }
        v = max(v, carry);
        __syncthreads();
        if (g <= n_groups) offsets[g] = v;
        carry = top;
    }
}

struct Plan {
    int passes, bits;      // digits and bits per digit
    int rounds;
    int64_t nblk;
    int64_t hist, totals, ka, ia, kb, ib, kout, bytes;     // byte offsets in the workspace
};

static Plan plan_for(int64_t n, int64_t n_groups) {
    Plan p = {};
    int b = 1;
    while (b < 31 && (((int64_t)1 << b) <= n_groups)) ++b;      // keys 0 .. n_groups
    const int most = n <= SMALL_N ? 8 : MAX_BITS;
    p.passes = (b + most - 1) / most;
    p.bits = (b + p.passes - 1) / p.passes;
    // rows a thread takes: few where the blocks would not fill the chip otherwise (786 432 rows: 4 rounds 15 us, 8 rounds 17)
    p.rounds = n < ((int64_t)1 << 20) ? 4 : 16;
    p.nblk = (n + p.rounds * BLOCK_THREADS - 1) / (p.rounds * BLOCK_THREADS);
    int64_t at = 0;
    auto take = [&](int64_t ints) {
        const int64_t here = at;
        at += (ints * 4 + 255) / 256 * 256;
        return here;
    };
    if (n > SMALL_N) {
        p.hist = take(((int64_t)1 << p.bits) * p.nblk);
        p.totals = take((int64_t)1 << p.bits);
        if (p.passes > 1) { p.ka = take(n); p.ia = take(n); }
        if (p.passes > 2) { p.kb = take(n); p.ib = take(n); }
    }
    if (p.passes > 1) p.kout = take(n);
    p.bytes = at < 256 ? 256 : at;
    return p;
}

static inline bool sizes_ok(int64_t n, int64_t n_groups) {
    return n >= 0 && n <= MAX_ROWS && n_groups >= 1 && n_groups <= MAX_GROUPS;
}

}  // namespace grp
}  // namespace nerf

extern "C" int64_t nerf_group_rows_workspace_bytes(int64_t n, int64_t n_groups) {
    if (!nerf::grp::sizes_ok(n, n_groups)) return NERF_E_SHAPE;
    return nerf::grp::plan_for(n, n_groups).bytes;
}

int64_t nerf::grp::workspace_bytes(int64_t n, int64_t n_groups) { return plan_for(n, n_groups).bytes; }

int nerf::grp::launch_group_rows(int64_t n, const void* ids, int id_bytes, int64_t n_groups, int32_t* order, int32_t* offsets,
                                 int32_t* tile_base, int32_t* keys, void* workspace, hipStream_t st) {
    const Plan p = plan_for(n, n_groups);
    char* ws = (char*)workspace;
    int32_t* kout = keys ? keys : (p.passes > 1 ? (int32_t*)(ws + p.kout) : nullptr);
    const int G = (int)n_groups;
    if (n <= SMALL_N) {
        if (id_bytes == 8)
            hipLaunchKernelGGL(small_kernel<int64_t>, dim3(1), dim3(SMALL_THREADS), 0, st, (int)n, (const int64_t*)ids, G, p.passes,
                               p.bits, order, offsets, tile_base, kout);
        else
            hipLaunchKernelGGL(small_kernel<int32_t>, dim3(1), dim3(SMALL_THREADS), 0, st, (int)n, (const int32_t*)ids, G, p.passes,
                               p.bits, order, offsets, tile_base, kout);
    } else {
        int32_t *hist = (int32_t*)(ws + p.hist), *totals = (int32_t*)(ws + p.totals);
        int32_t *ka = (int32_t*)(ws + p.ka), *ia = (int32_t*)(ws + p.ia), *kb = (int32_t*)(ws + p.kb), *ib = (int32_t*)(ws + p.ib);
        const dim3 grid((unsigned)p.nblk), block(BLOCK_THREADS), scan_grid(((1u << p.bits) + SCAN_DIGITS - 1) / SCAN_DIGITS);
        const int nblk = (int)p.nblk;
        const unsigned lds_hist = 4u << p.bits, lds_scatter = (BLOCK_THREADS / 64 + 1) * (4u << p.bits);
        const int32_t *kin = nullptr, *iin = nullptr;
        for (int pass = 0; pass < p.passes; ++pass) {
            const bool last = pass == p.passes - 1;
            int32_t* ko = last ? kout : (pass & 1 ? kb : ka);
            int32_t* io = last ? order : (pass & 1 ? ib : ia);
            const int shift = pass * p.bits;
#define NERF_PASS(ID, ROUNDS, SRC)                                                                                                   \
    do {                                                                                                                             \
        hipLaunchKernelGGL((hist_kernel<ID, ROUNDS>), grid, block, lds_hist, st, n, (const ID*)(SRC), (unsigned)G, shift, p.bits,     \
                           hist);                                                                                                    \
        hipLaunchKernelGGL(colscan_kernel, scan_grid, dim3(SCAN_DIGITS * 64), 0, st, nblk, 1 << p.bits, hist, totals);                \
        hipLaunchKernelGGL((scatter_kernel<ID, ROUNDS>), grid, block, lds_scatter, st, n, (const ID*)(SRC), iin, (unsigned)G, shift,  \
                           p.bits, hist, totals, ko, io, p.passes == 1 ? 1 : 0, offsets, tile_base);                            \
    } while (0)
#define NERF_PASS_R(ID, SRC)                                        \
    do {                                                            \
        if (p.rounds == 4) NERF_PASS(ID, 4, SRC);                   \
        else NERF_PASS(ID, 16, SRC);                                \
    } while (0)
            if (pass > 0) NERF_PASS_R(int32_t, kin);
            else if (id_bytes == 8) NERF_PASS_R(int64_t, ids);
            else NERF_PASS_R(int32_t, ids);
#undef NERF_PASS_R
#undef NERF_PASS
            kin = ko;
            iin = io;
        }
    }
    if (p.passes > 1) {
        hipLaunchKernelGGL(offsets_kernel, dim3((unsigned)((n_groups + BLOCK_THREADS) / BLOCK_THREADS)), dim3(BLOCK_THREADS), 0, st, n,
                           kout, G, offsets);
        if (tile_base) hipLaunchKernelGGL(tile_base_kernel, dim3(1), dim3(SMALL_THREADS), 0, st, (int)n, G, offsets, tile_base);
    }
    return nerf_launch_status();
}

extern "C" int nerf_group_rows(int64_t n, const void* ids, int id_bytes, int64_t n_groups, int32_t* order, int32_t* offsets,
                               int32_t* tile_base, void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace nerf::grp;
    NERF_REQUIRE(sizes_ok(n, n_groups), NERF_E_SHAPE);
    NERF_REQUIRE(id_bytes == 4 || id_bytes == 8, NERF_E_DTYPE);
    if (n == 0) return NERF_OK;
    NERF_REQUIRE(ids && order && offsets && workspace, NERF_E_NULL);
    NERF_REQUIRE(nerf_aligned(ids, (uintptr_t)id_bytes) && nerf_aligned(workspace, 256), NERF_E_ALIGN);
    NERF_REQUIRE(workspace_bytes >= plan_for(n, n_groups).bytes, NERF_E_WORKSPACE);
    return launch_group_rows(n, ids, id_bytes, n_groups, order, offsets, tile_base, nullptr, workspace, (hipStream_t)stream);
}

extern "C" int nerf_group_offsets(int64_t n, int64_t n_groups, const int32_t* offsets_in, int32_t* offsets, int32_t* tile_base,
                                  void* stream) {
    using namespace nerf::grp;
    NERF_REQUIRE(sizes_ok(n, n_groups), NERF_E_SHAPE);
    if (n == 0) return NERF_OK;
    NERF_REQUIRE(offsets_in && offsets && tile_base, NERF_E_NULL);
    hipStream_t st = (hipStream_t)stream;
    hipLaunchKernelGGL(clean_offsets_kernel, dim3(1), dim3(SMALL_THREADS), 0, st, (int)n, (int)n_groups, offsets_in, offsets);
    hipLaunchKernelGGL(tile_base_kernel, dim3(1), dim3(SMALL_THREADS), 0, st, (int)n, (int)n_groups, offsets, tile_base);
    return nerf_launch_status();
}
