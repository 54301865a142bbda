// Embedding lookup with scaling, out[n] = scale * table[token_n], and its gradient by sorted tokens,
// d_table[v] = scale * sum over the n with token_n = v of d_out[n]  (a token outside [0, V): a zero row, no gradient).
//
// Up to kFewMost tokens each row of the table looks for its own.  Beyond, the gradient sorts (token, n) stably, so that a token's rows
// stand together in ascending n; one wave sums the rows of a fixed number of sorted places and writes the runs of equal tokens that lie
// inside, runs that reach over a border leave fp32 shares that a second launch adds in order.  No float atomics: the result does not
// depend on the launch, and a token that holds a large share of all places is summed by as many waves as its places fill.  Both
// directions are bound by memory.
#include <type_traits>

#include "e4m3.h"

namespace phonlp {

template <class I>
__device__ __forceinline__ int token_key(const I *tokens, long n, int V) {  // V: no row
    const I t = tokens[n];
    return t >= 0 && t < (I)V ? (int)t : V;
}

// A lane takes VEC <= E neighbouring columns of a row; one that would reach behind the row's end takes its last VEC, some of them with its
// neighbour, and both then hold and write the same values.  (A branch for every column of every row takes longer than the loads: 512 rows
// on one wave, eight columns of bf16 a lane, 247 us against 121.)
//
// A wave takes sixteen tokens and a slab of 64 * VEC columns (blockIdx.y): one load for the tokens, a lane each, sixteen rows in flight.
// Lanes behind a row's end stay with the others: the tokens are read from all sixteen lanes.
template <int VEC, class T, class I>
__global__ __launch_bounds__(256) void embedding_rows_kernel(const T *table, long ld, const I *tokens, int N, int V, int E, float scale,
                                                             T *out) {
    constexpr int ROWS = 16;
    typedef typename Vec<T, VEC>::type Vt;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), from = (blockIdx.y * 64 + lane) * VEC,
              col = min(from, E - VEC);  // at a row's end some columns twice, the same values
    const long n0 = (blockIdx.x * 4L + wave) * ROWS;
    if (n0 >= N) return;  // the whole wave
    const int rows = (int)min((long)ROWS, N - n0), held = token_key(tokens, n0 + min(lane, rows - 1), V);
    int key[ROWS];
#pragma unroll
    for (int u = 0; u < ROWS; ++u) key[u] = __builtin_amdgcn_readlane(held, u);
    if (from >= E) return;
    Vt v[ROWS];
#pragma unroll
    for (int u = 0; u < ROWS; ++u) v[u] = *reinterpret_cast<const Vt *>(table + (key[u] < V ? key[u] : 0) * ld + col);
#pragma unroll
    for (int u = 0; u < ROWS; ++u) {
        Vt o;
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = key[u] < V ? (T)((float)v[u][i] * scale) : (T)0.f;
        if (u < rows) *reinterpret_cast<Vt *>(out + (n0 + u) * E + col) = o;
    }
}

// ---- sorting, few tokens: a token's place is the number of (token, n) pairs before its own.  N^2 comparisons in one launch; a workgroup
// places 32 tokens, 32 threads a token count a share of the others each.  A gradient of eight columns takes 17 us for 4096 tokens and 21
// for 8192, against 25 and 24 by radix passes; for 12288 37 against 26.
constexpr int kPlaceThreads = 1024;
template <class I>
__global__ __launch_bounds__(kPlaceThreads) void embedding_place_kernel(const I *tokens, int N, int V, int *order, int *sorted) {
    constexpr int TILE = 4096, THREADS = kPlaceThreads, PARTS = THREADS / 32, EACH = TILE / THREADS;
    __shared__ __attribute__((aligned(16))) int keys[TILE];
    __shared__ int counts[PARTS][32];
    const int own = threadIdx.x & 31, part = threadIdx.x >> 5, n0 = blockIdx.x * 32, n = n0 + own;
    const int key = n < N ? token_key(tokens, n, V) : 0;
    int count = 0;
    for (int base = 0; base < N; base += TILE) {
        __syncthreads();
        I t[EACH];
#pragma unroll
        for (int i = 0; i < EACH; ++i) t[i] = tokens[min(base + i * THREADS + (int)threadIdx.x, N - 1)];
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            const int at = i * THREADS + threadIdx.x;
            keys[at] = base + at >= N ? 0x7FFFFFFF : t[i] >= 0 && t[i] < (I)V ? (int)t[i] : V;
        }
        __syncthreads();
        // this thread's share of them, 32 at a time: equal ones count if they stand before n
#pragma unroll 1
        for (int i = part * (TILE / PARTS); i < (part + 1) * (TILE / PARTS) && base + i < N; i += 32) {
            const int first = n0 - base - i, bound = key + (first > 0);  // first = 0: this workgroup's own 32
#pragma unroll
            for (int j = 0; j < 32; j += 4) {
                const int4 k = *reinterpret_cast<const int4 *>(keys + i + j);
                if (first) count += (k.x < bound) + (k.y < bound) + (k.z < bound) + (k.w < bound);
                else count += (k.x < key + (j < own)) + (k.y < key + (j + 1 < own)) + (k.z < key + (j + 2 < own)) + (k.w < key + (j + 3 < own));
            }
        }
    }
    counts[part][own] = count;
    __syncthreads();
    if (part == 0 && n < N) {
        int place = 0;
#pragma unroll
        for (int i = 0; i < PARTS; ++i) place += counts[i][own];
        order[place] = n;
        sorted[place] = key;
    }
}

// ---- sorting, many tokens: stable radix passes of eight bits in at most 256 tiles of pairs, two launches a pass.
template <class I>
__device__ __forceinline__ int sort_key(const I *tokens, const int *keys, long n, int V) {
    return keys ? keys[n] : token_key(tokens, n, V);
}

// counts[tile][digit]
template <class I>
__global__ __launch_bounds__(256) void embedding_count_kernel(const I *tokens, const int *keys, int N, int V, int shift, int tile, int *counts) {
    __shared__ int bins[256];
    bins[threadIdx.x] = 0;
    __syncthreads();
    const long base = (long)blockIdx.x * tile;
    for (int i = threadIdx.x; i < tile && base + i < N; i += 1024) {  // four loads in flight
        int key[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) key[u] = sort_key(tokens, keys, min(base + i + u * 256, N - 1L), V);
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (base + i + u * 256 < N) atomicAdd(&bins[key[u] >> shift & 255], 1);
    }
    __syncthreads();
    counts[blockIdx.x * 256 + threadIdx.x] = bins[threadIdx.x];
}

template <class I>
__global__ __launch_bounds__(256) void embedding_scatter_kernel(const I *tokens, const int *keys, const int *index, int N, int V, int shift,
                                                                int tile, const int *counts, int *keys_out, int *index_out) {
    __shared__ int at[4][256];  // the next place of each wave's pairs of a digit
    __shared__ int totals[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tiles = gridDim.x;
    const long base = (long)blockIdx.x * tile + wave * (tile / 4);
#pragma unroll
    for (int w = 0; w < 4; ++w) at[w][threadIdx.x] = 0;
    __syncthreads();
    // four of the wave's pairs per lane at a time: those of the tile's first (and most often only) 256 stay in registers
    int key[4], from[4];
    auto read = [&](int r) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const long n = min(base + r + u * 64 + lane, N - 1L);
            key[u] = sort_key(tokens, keys, n, V);
            from[u] = index ? index[n] : (int)n;
        }
    };
    for (int r = tile / 4 - 256; r >= 0; r -= 256) {
        read(r);
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (base + r + u * 64 + lane < N) atomicAdd(&at[wave][key[u] >> shift & 255], 1);
    }
    // this thread's digit: the pairs of smaller digits, and those of its own in the tiles before
    int total = 0, before = 0;
#pragma unroll 8
    for (int t = 0; t < tiles; ++t) {
        const int c = counts[t * 256 + threadIdx.x];
        total += c;
        before += t < (int)blockIdx.x ? c : 0;
    }
    int scan = total;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(scan, d);
        if (lane >= d) scan += o;
    }
    if (lane == 63) totals[wave] = scan;
    __syncthreads();
    int place = before + scan - total;
#pragma unroll
    for (int w = 0; w < 4; ++w) place += w < wave ? totals[w] : 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const int c = at[w][threadIdx.x];
        at[w][threadIdx.x] = place;
        place += c;
    }
    __syncthreads();
    for (int r = 0; r < tile / 4; r += 256) {
        if (r) read(r);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const bool in = base + r + u * 64 + lane < N;
            const int digit = key[u] >> shift & 255;
            // the lanes that hold a pair of the same digit
            unsigned long long same = __ballot(in);
#pragma unroll
            for (int b = 0; b < 8; ++b) {
                const unsigned long long set = __ballot(digit >> b & 1);
                same &= digit >> b & 1 ? set : ~set;
            }
            const int rank = __popcll(same & ((1ull << lane) - 1));
            int first = 0;
            if (in) first = at[wave][digit];
            __builtin_amdgcn_wave_barrier();
            if (in) {
                keys_out[first + rank] = key[u];
                index_out[first + rank] = from[u];
                if (rank == 0) at[wave][digit] = first + __popcll(same);
            }
            __builtin_amdgcn_wave_barrier();
        }
    }
}

// ---- sums
// The first place >= lo whose token is >= key.
__device__ __forceinline__ int lower_bound(const int *sorted, int lo, int hi, int key) {
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sorted[mid] < key) lo = mid + 1;
        else hi = mid;
    }
    return lo;
}

// The same by a whole wave, for a key that all its lanes have: 64 places a step.
__device__ __forceinline__ int lower_bound_wave(const int *sorted, int n, int key, int lane) {
    int lo = 0, hi = n;
    while (lo < hi) {
        const int step = ceil_div(hi - lo, 64), at = lo + (lane + 1) * step - 1;
        const int less = __popcll(__ballot(at < hi && sorted[min(at, hi - 1)] < key));
        hi = min(hi, lo + (less + 1) * step - 1);
        lo += less * step;
    }
    return lo;
}

template <class TO, int VEC>
__device__ __forceinline__ void store_row(TO *p, const float (&v)[VEC], float scale) {
    typename Vec<TO, VEC>::type t;
#pragma unroll
    for (int i = 0; i < VEC; ++i) t[i] = (TO)(v[i] * scale);
    *reinterpret_cast<typename Vec<TO, VEC>::type *>(p) = t;
}

struct SumArgs {
    const void *d_out;
    void *d_table;
    float *shares;  // [chunks][2][E]: the sum of a chunk's first run that began before it, of its last run that goes on behind it
    const int *order, *sorted;
    long ld, row0;  // row0: the table's first row of this launch
    int N, V, E, R, chunks, sum_blocks;
    float scale;
};

// Few tokens, no sort: a workgroup owns `rows` <= 64 rows of the table (few, where the table is small: a row's tokens come one after the
// other) and a slab of columns.  Each of its four waves takes a quarter of the tokens, two a lane at most, and adds those of a row in
// ascending n; a row that several waves have tokens of is the sum of their shares in ascending order, one without tokens is zeros.
// One launch in place of three: 64000 x 768 bf16, 37 tokens 16.6 us against 20.3 by sorted tokens, 512 tokens 19.3 against 22.5; 24 x 100
// fp32, 512 tokens 4.2 against 13.5; at worst, 512 times the same token of 1000 x 768 bf16, 30 against 15.
constexpr int kFewMost = 512;
template <int VEC, class T, class TO, class I>
__global__ __launch_bounds__(256) void embedding_few_kernel(const T *d, long ld, const I *tokens, int N, int V, int E, long base, int rows,
                                                            float scale, TO *table) {
    constexpr int UNROLL = 16;
    typedef typename Vec<T, VEC>::type Vt;
    __shared__ float shares[4][64 * VEC];
    __shared__ unsigned there[4][2];  // of each wave, the rows that it has tokens of
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), from = (blockIdx.y * 64 + lane) * VEC,
              col = min(from, E - VEC), each = ceil_div(N, 4), first = wave * each, mine = min(each, N - first);
    const long row0 = base + (long)blockIdx.x * rows;
    const int have = (int)min((long)rows, V - row0);
    if (threadIdx.x < 8) there[threadIdx.x >> 1][threadIdx.x & 1] = 0;
    __syncthreads();
    int at[2];  // which of the rows, for this wave's tokens lane and 64 + lane
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int n = h * 64 + lane, key = token_key(tokens, min(first + n, N - 1), V);
        const long r = key - row0;
        at[h] = n < mine && key < V && r >= 0 && r < have ? (int)r : -1;
        if (at[h] >= 0) atomicOr(&there[wave][at[h] >> 5], 1u << (at[h] & 31));
    }
    __syncthreads();
    unsigned long long one = 0, more = 0, own = 0;  // rows with tokens of one wave or more, of two or more, of this one
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const unsigned long long m = there[w][0] | (unsigned long long)there[w][1] << 32;
        more |= one & m;
        one |= m;
        if (w == wave) own = m;
    }
    auto add = [&](int r, float (&s)[VEC]) {  // this wave's rows of token row0 + r
        unsigned long long low = __ballot(at[0] == r), high = __ballot(at[1] == r);
        while (low | high) {
            int n[UNROLL], count = 0;
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const bool any = low | high;
                const unsigned long long m = low ? low : high, rest = m & (m - 1);
                n[u] = any ? first + (low ? 0 : 64) + __ffsll(m) - 1 : n[u ? u - 1 : 0];
                high = low ? high : rest;
                low = low ? rest : 0;
                count += any;
            }
            Vt v[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) v[u] = *reinterpret_cast<const Vt *>(d + n[u] * ld + col);
#pragma unroll
            for (int u = 0; u < UNROLL; ++u)
#pragma unroll
                for (int i = 0; i < VEC; ++i) s[i] += u < count ? (float)v[u][i] : 0.f;
        }
    };
    TO *out = table + row0 * E + col;
    const bool in = from < E;
    if (in) {
        const float zero[VEC] = {};
        for (unsigned long long rest = ~one & (~0ull >> (64 - have)) & 0x1111111111111111ull << wave; rest; rest &= rest - 1)
            store_row<TO, VEC>(out + (long)(__ffsll(rest) - 1) * E, zero, 0.f);
    }
    for (unsigned long long rest = own & ~more; rest; rest &= rest - 1) {
        const int r = __ffsll(rest) - 1;
        float s[VEC] = {};
        add(r, s);
        if (in) store_row<TO, VEC>(out + (long)r * E, s, scale);
    }
    for (unsigned long long rest = more; rest; rest &= rest - 1) {  // all four waves
        const int r = __ffsll(rest) - 1;
        float s[VEC] = {};
        add(r, s);
#pragma unroll
        for (int i = 0; i < VEC; ++i) shares[wave][i * 64 + lane] = s[i];
        __syncthreads();
        if (wave == 0) {
#pragma unroll
            for (int w = 1; w < 4; ++w)
#pragma unroll
                for (int i = 0; i < VEC; ++i) s[i] += shares[w][i * 64 + lane];
            if (in) store_row<TO, VEC>(out + (long)r * E, s, scale);
        }
        __syncthreads();
    }
}

// blockIdx.y: a slab of 64 * VEC columns.  blockIdx.x < sum_blocks: a wave per chunk of R sorted places, sixteen rows in flight; behind
// them (first slab only): a wave per 16 rows of the table, which writes zeros where no token points (64 tokens, 64000 x 768
// bf16: 22.3 us with a search per row, 21.2 with one per 16).
template <int VEC, class T, class TO>
__global__ __launch_bounds__(256) void embedding_sum_kernel(SumArgs a) {
    constexpr int UNROLL = 16;
    typedef typename Vec<T, VEC>::type Vt;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    TO *table = (TO *)a.d_table;
    if ((int)blockIdx.x >= a.sum_blocks) {
        if (blockIdx.y) return;
        const long row0 = a.row0 + ((long)(blockIdx.x - a.sum_blocks) * 4 + wave) * 16;
        if (row0 >= a.V) return;
        unsigned long long rows = (1ull << min(a.V - row0, 16L)) - 1;  // those that no token points at
        const int from = lower_bound_wave(a.sorted, a.N, (int)row0, lane);
        const int key = from + lane < a.N ? a.sorted[from + lane] : 0x7FFFFFFF;
        if (__builtin_amdgcn_readlane(key, 63) >= row0 + 16) {  // the next 64 places hold all of their tokens
#pragma unroll
            for (int r = 0; r < 16; ++r) rows &= ~((unsigned long long)(__ballot(key == row0 + r) != 0) << r);
        } else {
            bool there = false;
            if (lane < 16) {
                const int at = lower_bound(a.sorted, from, a.N, (int)row0 + lane);
                there = at < a.N && a.sorted[at] == row0 + lane;
            }
            rows &= ~__ballot(there);
        }
        const float zero[VEC] = {};
        while (rows) {
            const int r = __ffsll(rows) - 1;
            rows &= rows - 1;
            for (int c = lane * VEC; c < a.E; c += 64 * VEC) store_row<TO, VEC>(table + (row0 + r) * a.E + min(c, a.E - VEC), zero, 0.f);
        }
        return;
    }
    const int chunk = blockIdx.x * 4 + wave, from = (blockIdx.y * 64 + lane) * VEC, col = min(from, a.E - VEC);
    if (chunk >= a.chunks) return;
    const int first = chunk * a.R, last = min(first + a.R, a.N);
    const T *d = (const T *)a.d_out;
    bool head = first > 0 && a.sorted[first - 1] == a.sorted[first];  // the first run began before
    float s[VEC] = {};
    for (int p = first; p < last; p += UNROLL) {
        // lane u holds place p + u
        const int at = p + lane, row = a.order[min(at, last - 1)], key = at < a.N ? a.sorted[at] : -1;
        Vt v[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) v[u] = *reinterpret_cast<const Vt *>(d + (long)__builtin_amdgcn_readlane(row, u) * a.ld + col);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            if (p + u >= last) break;
#pragma unroll
            for (int i = 0; i < VEC; ++i) s[i] += (float)v[u][i];
            const int k = __builtin_amdgcn_readlane(key, u);
            const bool ends = __builtin_amdgcn_readlane(key, u + 1) != k;
            if (!ends && p + u + 1 < last) continue;
            if (from < a.E && k < a.V) {
                if (ends && !head) store_row<TO, VEC>(table + (long)k * a.E + col, s, a.scale);
                else store_row<float, VEC>(a.shares + ((long)chunk * 2 + (head ? 0 : 1)) * a.E + col, s, 1.f);
            }
            head = false;
#pragma unroll
            for (int i = 0; i < VEC; ++i) s[i] = 0.f;
        }
    }
}

// Runs that go on behind the chunk they begin in: their shares, in order.  A workgroup looks at eight chunks, a chunk per lane; runs of
// up to 17 shares are summed by a wave each, longer ones by all eight waves, an eighth of the shares each.
template <int VEC, class TO>
__global__ __launch_bounds__(512) void embedding_join_kernel(SumArgs a) {
    constexpr int UNROLL = VEC == 8 ? 8 : 16, FEW = 16;
    __shared__ float sums[8][64 * VEC];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), from = (blockIdx.y * 64 + lane) * VEC,
              col = min(from, a.E - VEC), mine = blockIdx.x * 8 + lane;
    const bool in = from < a.E;
    auto reaches = [&](int chunk, int k) {  // the first place of `chunk` still holds k
        const long p = (long)chunk * a.R;
        return (p < a.N) & (a.sorted[min(p, (long)a.N - 1)] == k);
    };
    int key = a.V, count = 1;  // shares behind the chunk's own, at most FEW
    if (lane < 8 && mine < a.chunks - 1) {
        const int first = mine * a.R, k = a.sorted[first + a.R - 1];
        const bool began_before = a.sorted[first] == k && first > 0 && a.sorted[first - 1] == k;
        if (k < a.V && reaches(mine + 1, k) && !began_before) {
            key = k;
#pragma unroll
            for (int i = 2; i <= FEW; ++i) count += reaches(mine + i, k);
        }
    }
    auto add = [&](int chunk, int lo, int hi, float (&s)[VEC]) {  // shares lo .. hi - 1: the chunk's last run, then the next chunks' first
        for (int c = lo; c < hi; c += UNROLL) {
            typedef typename Vec<float, VEC>::type Vf;
            Vf v[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int k = min(c + u, hi - 1);
                v[u] = *reinterpret_cast<const Vf *>(a.shares + ((long)(chunk + k) * 2 + (k ? 0 : 1)) * a.E + col);
            }
#pragma unroll
            for (int u = 0; u < UNROLL; ++u)
#pragma unroll
                for (int i = 0; i < VEC; ++i)
                    if (c + u < hi) s[i] += v[u][i];
        }
    };
    auto store = [&](int k, const float (&s)[VEC]) { store_row<TO, VEC>((TO *)a.d_table + (long)k * a.E + col, s, a.scale); };
    int turn = 0;
    for (unsigned long long runs = __ballot(key < a.V); runs; runs &= runs - 1) {
        const int l = __ffsll(runs) - 1, chunk = blockIdx.x * 8 + l, k = __builtin_amdgcn_readlane(key, l);
        int n = __builtin_amdgcn_readlane(count, l) + 1;
        if (n > FEW) {  // how many of the chunks left it reaches: 64 of them far apart, then the 64 (or more) in between, and so on
            for (int apart = ceil_div(a.chunks - chunk - n, 64); apart > 0; apart = apart > 1 ? ceil_div(apart, 64) : 0)
                n += __popcll(__ballot(reaches(chunk + n + lane * apart + apart - 1, k))) * apart;
        }
        float s[VEC] = {};
        if (n <= FEW + 1) {
            if ((turn++ & 7) == wave && in) {
                add(chunk, 0, n, s);
                store(k, s);
            }
            continue;
        }
        const int per = ceil_div(n, 8);
        if (in) add(chunk, wave * per, min(wave * per + per, n), s);
#pragma unroll
        for (int i = 0; i < VEC; ++i) sums[wave][i * 64 + lane] = s[i];
        __syncthreads();
        if (wave == 0 && in) {
#pragma unroll
            for (int w = 1; w < 8; ++w)
#pragma unroll
                for (int i = 0; i < VEC; ++i) s[i] += sums[w][i * 64 + lane];
            store(k, s);
        }
        __syncthreads();
    }
}

// Tokens or rows of the table that one launch covers: a grid holds less than 2^32 threads.
constexpr int kLaunchMost = 1 << 29;
constexpr int kPlaceMost = 8192;  // tokens sorted by counting (above)
struct EmbeddingPlan {
    int R, chunks, tile, tiles;  // places of one wave; pairs of a sorting tile
    size_t pairs, shares, counts, total;
};
static EmbeddingPlan plan_embedding(int N, int E) {
    EmbeddingPlan p;
    p.R = ceil_div(ceil_div(N, 4096), 16) * 16;  // enough waves to fill the chip, few enough shares to join
    p.chunks = ceil_div(N, p.R);
    p.tile = ceil_div(ceil_div(N, 256), 1024) * 1024;
    p.tiles = ceil_div(N, p.tile);
    p.pairs = align_up((size_t)N * 4, 256);
    p.shares = align_up((size_t)p.chunks * 2 * E * 4, 256);
    const bool radix = N > kPlaceMost;
    p.counts = radix ? align_up((size_t)p.tiles * 256 * 4, 256) : 0;
    p.total = p.pairs * (radix ? 4 : 2) + p.shares + p.counts;
    return p;
}

template <class I>
static int sort_tokens(const I *tokens, int N, int V, const EmbeddingPlan &pl, char *ws, int **order, int **sorted, hipStream_t st) {
    ProfScope ps("embedding_sort", st);
    int *k[2] = {(int *)ws, (int *)(ws + pl.pairs)};
    if (N <= kPlaceMost) {
        hipLaunchKernelGGL((embedding_place_kernel<I>), dim3(ceil_div(N, 32)), dim3(kPlaceThreads), 0, st, tokens, N, V, k[0], k[1]);
        *order = k[0];
        *sorted = k[1];
        return check_launch("embedding_place_kernel");
    }
    int *keys[2] = {k[0], k[1]}, *index[2] = {(int *)(ws + 2 * pl.pairs), (int *)(ws + 3 * pl.pairs)};
    int *counts = (int *)(ws + 4 * pl.pairs + pl.shares);
    const int *from_keys = nullptr, *from_index = nullptr;
    int now = 0;
    for (int shift = 0; shift == 0 || (shift < 31 && (V >> shift) > 0); shift += 8, now ^= 1) {  // keys 0 .. V
        hipLaunchKernelGGL((embedding_count_kernel<I>), dim3(pl.tiles), dim3(256), 0, st, tokens, from_keys, N, V, shift, pl.tile, counts);
        hipLaunchKernelGGL((embedding_scatter_kernel<I>), dim3(pl.tiles), dim3(256), 0, st, tokens, from_keys, from_index, N, V, shift,
                           pl.tile, counts, keys[now], index[now]);
        const int rc = check_launch("embedding_scatter_kernel");
        if (rc) return rc;
        from_keys = keys[now];
        from_index = index[now];
    }
    *sorted = keys[now ^ 1];
    *order = index[now ^ 1];
    return PHONLP_OK;
}

template <int VEC, class T, class TO>
static int sum_rows(SumArgs a, hipStream_t st) {
    const int slabs = ceil_div(a.E, 64 * VEC);
    a.sum_blocks = ceil_div(a.chunks, 4);
    {
        ProfScope ps("embedding_sum", st);
        do {
            const int rows = (int)(a.V - a.row0 < kLaunchMost ? a.V - a.row0 : kLaunchMost);
            hipLaunchKernelGGL((embedding_sum_kernel<VEC, T, TO>), dim3(a.sum_blocks + ceil_div(rows, 64), slabs), dim3(256), 0, st, a);
            const int rc = check_launch("embedding_sum_kernel");
            if (rc) return rc;
            a.sum_blocks = 0;  // the sums are made
        } while ((a.row0 += kLaunchMost) < a.V);
    }
    if (a.chunks == 1) return PHONLP_OK;
    ProfScope ps("embedding_join", st);
    hipLaunchKernelGGL((embedding_join_kernel<VEC, TO>), dim3(ceil_div(a.chunks - 1, 8), slabs), dim3(512), 0, st, a);
    return check_launch("embedding_join_kernel");
}

template <int VEC, class T, class TO, class I>
static int few_rows(const SumArgs &a, const I *tokens, hipStream_t st) {
    ProfScope ps("embedding_few", st);
    const int rows = a.V >= 65536 ? 64 : ceil_div(a.V, 1024);  // of a workgroup: some thousand of them a slab
    for (long base = 0; base < a.V; base += kLaunchMost) {
        const int most = (int)(a.V - base < kLaunchMost ? a.V - base : kLaunchMost);
        hipLaunchKernelGGL((embedding_few_kernel<VEC, T, TO, I>), dim3(ceil_div(most, rows), ceil_div(a.E, 64 * VEC)), dim3(256), 0, st,
                           (const T *)a.d_out, a.ld, tokens, a.N, a.V, a.E, base, rows, a.scale, (TO *)a.d_table);
        const int rc = check_launch("embedding_few_kernel");
        if (rc) return rc;
    }
    return PHONLP_OK;
}

// Calls f with the widest vector of T (16 bytes, 4 elements or one) that a row of E holds.
template <class T, class F>
static int with_vec(int E, F &&f) {
    if (E >= 16 / (int)sizeof(T)) return f(std::integral_constant<int, 16 / (int)sizeof(T)>{});
    if (E >= 4) return f(std::integral_constant<int, 4>{});
    return f(std::integral_constant<int, 1>{});
}

}  // namespace phonlp

using namespace phonlp;

extern "C" int phonlp_embedding_rows(const void *table, int type, long ld, const void *tokens, int tokens_are_int64, int N, int V, int E,
                                     float scale, void *out, void *stream) {
    if (!table || !tokens || !out || !type_ok(type) || N <= 0 || N > (1 << 30) || V <= 0 || E <= 0 || E > (1 << 22) || ld < E ||
        V == 0x7FFFFFFF)
        return fail(PHONLP_ERR_SHAPE, "embedding_rows: bad argument");
    if ((uintptr_t)table % type_bytes(type) || (uintptr_t)out % type_bytes(type) || (uintptr_t)tokens % (tokens_are_int64 ? 8 : 4))
        return fail(PHONLP_ERR_SHAPE, "embedding_rows: table, tokens and out must have their types' alignment");
    hipStream_t st = as_stream(stream);
    ProfScope ps("embedding_rows", st);
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        return with_vec<T>(E, [&](auto vec) {
            constexpr int VEC = decltype(vec)::value;
            auto launch = [&](auto *tok) {
                using I = std::remove_cv_t<std::remove_pointer_t<decltype(tok)>>;
                for (long n = 0; n < N; n += kLaunchMost) {
                    const int most = (int)(N - n < kLaunchMost ? N - n : kLaunchMost);
                    hipLaunchKernelGGL((embedding_rows_kernel<VEC, T, I>), dim3(ceil_div(most, 64), ceil_div(E, 64 * VEC)), dim3(256), 0, st,
                                       (const T *)table, ld, tok + n, most, V, E, scale, (T *)out + n * E);
                    const int rc = check_launch("embedding_rows_kernel");
                    if (rc) return rc;
                }
                return (int)PHONLP_OK;
            };
            return tokens_are_int64 ? launch((const long *)tokens) : launch((const int *)tokens);
        });
    });
}

extern "C" size_t phonlp_embedding_rows_grad_ws_bytes(int N, int E) {
    return N > 0 && N <= (1 << 30) && E > 0 && E <= (1 << 22) ? plan_embedding(N, E).total : 0;
}

extern "C" int phonlp_embedding_rows_grad(const void *d_out, int type, long ld, const void *tokens, int tokens_are_int64, int N, int V,
                                          int E, float scale, void *d_table, int table_type, void *ws, size_t ws_bytes, void *stream) {
    if (!d_out || !tokens || !d_table || !type_ok(type) || N <= 0 || N > (1 << 30) || V <= 0 || V == 0x7FFFFFFF || E <= 0 ||
        E > (1 << 22) || ld < E || (table_type != type && table_type != PHONLP_F32))
        return fail(PHONLP_ERR_SHAPE, "embedding_rows_grad: bad argument (d_table is of d_out's type or fp32)");
    if ((uintptr_t)d_out % type_bytes(type) || (uintptr_t)d_table % type_bytes(table_type) || (uintptr_t)tokens % (tokens_are_int64 ? 8 : 4))
        return fail(PHONLP_ERR_SHAPE, "embedding_rows_grad: d_out, tokens and d_table must have their types' alignment");
    if (!ws || ((uintptr_t)ws & 15) || ws_bytes < phonlp_embedding_rows_grad_ws_bytes(N, E))
        return fail(PHONLP_ERR_WORKSPACE, "embedding_rows_grad: workspace too small or not 16-byte aligned");
    hipStream_t st = as_stream(stream);
    const EmbeddingPlan pl = plan_embedding(N, E);
    SumArgs a = {d_out, d_table, nullptr, nullptr, nullptr, ld, 0, N, V, E, pl.R, pl.chunks, 0, scale};
    const bool few = N <= kFewMost, radix = N > kPlaceMost;
    if (!few) {
        int *order, *sorted;
        const int rc = tokens_are_int64 ? sort_tokens((const long *)tokens, N, V, pl, (char *)ws, &order, &sorted, st)
                                        : sort_tokens((const int *)tokens, N, V, pl, (char *)ws, &order, &sorted, st);
        if (rc) return rc;
        a.order = order;
        a.sorted = sorted;
        a.shares = (float *)((char *)ws + pl.pairs * (radix ? 4 : 2));
    }
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        return with_vec<T>(E, [&](auto vec) {
            constexpr int VEC = decltype(vec)::value;
            auto run = [&](auto to) {
                using TO = decltype(to);
                if (!few) return sum_rows<VEC, T, TO>(a, st);
                return tokens_are_int64 ? few_rows<VEC, T, TO>(a, (const long *)tokens, st) : few_rows<VEC, T, TO>(a, (const int *)tokens, st);
            };
            return table_type == PHONLP_F32 ? run(float{}) : run(T{});
        });
    });
}
