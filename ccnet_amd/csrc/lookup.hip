// Token lookup with scaling, and its gradient by sorted tokens.
//
//   y[t] = scale * W[id[t]]                      (ids outside [0, vocab): a row of zeros)
//   dW[v] = scale * sum over t with id[t] = v of dy[t], in rising t
//
// The gradient sorts (id, t) and then writes the row of every id that occurs once, in fp32, from a fixed tree over the id's run
// of sorted positions: no float atomics, so equal inputs give equal bits.  A run may hold one position or nearly all of them
// (the padding token of a batch of prompts), so runs are summed in three grains: single rows, whole aligned chunks of 64
// sorted positions and whole aligned chunks of 512 that lie inside one run (chunk_sum_kernel), joined by run_sum_kernel.
// Sorting keeps only a few of the 256 CUs busy: the others write the table's zeros meanwhile (Fill), rows that occur being
// overwritten afterwards.
#include "common.h"

#include <algorithm>

namespace {

typedef unsigned short bf16_t;

__device__ __forceinline__ void from_f32(float& d, float v) { d = v; }
__device__ __forceinline__ void from_f32(bf16_t& d, float v) { d = f32_to_bf16_bits(v); }

// Eight columns of a 512-column span a lane.  VECTOR: neighbours, rows 16-byte aligned and whole vectors long.  LOOSE: neighbours by
// accesses of the same width at the elements' alignment, the row's last columns one by one (50021 x 1023 bf16: lookup 49 -> 34.5 us,
// gradient 137 -> 100).  SPREAD, where all is fp32: every 64th column (78 us and 112, LOOSE 88 and 131).
enum Cols { VECTOR, LOOSE, SPREAD };
template <typename T, int L> struct Words;
template <> struct Words<float, VECTOR> { typedef f32x4 V; };
template <> struct Words<float, LOOSE> { typedef f32x4 __attribute__((aligned(4))) V; };
template <> struct Words<bf16_t, VECTOR> { typedef u32x4 V; };
template <> struct Words<bf16_t, LOOSE> { typedef u32x4 __attribute__((aligned(2))) V; };

// Eight columns as they lie in memory, so that many rows in flight cost no more registers than their bytes.  PAST: past the
// caches, for gradients that are larger than them (131k x 1024 bf16: 147 -> 132 us; 2464 x 1024, which stay in them: 50 -> 57).
template <typename T, int L, bool PAST = false> struct Raw;
template <int L, bool PAST> struct Raw<float, L, PAST> {
    static constexpr int DEEP = 8;
    f32x4 a, b;
    __device__ __forceinline__ void load(const float* row, int lane, int cols) {
        a = b = f32x4{0.f, 0.f, 0.f, 0.f};
        if constexpr (L == SPREAD) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (lane + 64 * j < cols) a[j] = row[lane + 64 * j];
                if (lane + 64 * (4 + j) < cols) b[j] = row[lane + 64 * (4 + j)];
            }
        } else {
            typedef typename Words<float, L>::V V;
            const int left = cols - lane * 8;
            const float* p = row + lane * 8;
            if (left >= (L == VECTOR ? 1 : 8)) {
                if constexpr (PAST) {
                    a = __builtin_nontemporal_load((const V*)p);
                    b = __builtin_nontemporal_load((const V*)(p + 4));
                } else {
                    a = *(const V*)p;
                    b = *(const V*)(p + 4);
                }
            } else if (L == LOOSE && left > 0) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (j < left) a[j] = p[j];
                    if (4 + j < left) b[j] = p[4 + j];
                }
            }
        }
    }
    __device__ __forceinline__ void get(float* f) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) { f[e] = a[e]; f[4 + e] = b[e]; }
    }
};
template <int L, bool PAST> struct Raw<bf16_t, L, PAST> {
    static constexpr int DEEP = 16;
    u32x4 a;
    __device__ __forceinline__ void load(const bf16_t* row, int lane, int cols) {
        typedef typename Words<bf16_t, L>::V V;
        const int left = cols - lane * 8;
        const bf16_t* p = row + lane * 8;
        a = u32x4{0u, 0u, 0u, 0u};
        if (left >= (L == VECTOR ? 1 : 8)) {
            if constexpr (PAST) a = __builtin_nontemporal_load((const V*)p);
            else a = *(const V*)p;
        } else if (L == LOOSE && left > 0) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                if (2 * w < left) a[w] = p[2 * w];
                if (2 * w + 1 < left) a[w] |= (unsigned)p[2 * w + 1] << 16;
            }
        }
    }
    __device__ __forceinline__ void get(float* f) const { unpack8(a, f); }
};
template <typename X>
__device__ __forceinline__ void add_raw(const X& x, float* acc) {
    float f[8];
    x.get(f);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] += f[e];
}
template <int L, typename T>
__device__ __forceinline__ void load8(const T* row, int lane, int cols, float* f) {
    Raw<T, L> x;
    x.load(row, lane, cols);
    x.get(f);
}
template <int L, typename T>
__device__ __forceinline__ void store8(T* row, int lane, int cols, const float* f) {
    if constexpr (L == SPREAD) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (lane + 64 * j < cols) row[lane + 64 * j] = f[j];
    } else {
        typedef typename Words<T, L>::V V;
        const int left = cols - lane * 8;
        T* p = row + lane * 8;
        if (left >= (L == VECTOR ? 1 : 8)) {
            if constexpr (sizeof(T) == 4) {
                *(V*)p = f32x4{f[0], f[1], f[2], f[3]};
                *(V*)(p + 4) = f32x4{f[4], f[5], f[6], f[7]};
            } else {
                *(V*)p = pack8(f);
            }
        } else if (L == LOOSE) {
#pragma unroll
            for (int j = 0; j < 7; ++j)
                if (j < left) from_f32(p[j], f[j]);
        }
    }
}

__device__ __forceinline__ long long id_at(const void* ids, int wide, long long t) {
    return wide ? ((const long long*)ids)[t] : (long long)((const int*)ids)[t];
}

// ------------------------------------------------------------------ lookup
// A wave per row, 512 columns at a time, 16 bytes a lane.  Bound by memory: every row written once, the rows of a table read from the
// caches where tokens repeat (50021 tokens of 49408, bf16 1024 -> bf16: 23.8 us, 4.3 TB/s written; 77 tokens: 2.6 us, of which the
// launch and two dependent loads are all).
template <typename TW, typename TO, int L>
__global__ __launch_bounds__(256) void lookup_kernel(const void* ids, int wide, int T, int vocab, const TW* table, long long ldt, int C,
                                                     float scale, TO* out, long long ldo) {
    const int lane = threadIdx.x & 63;
    const long long t = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= T) return;
    const long long id = id_at(ids, wide, t);
    const bool ok = id >= 0 && id < vocab;
    for (int c0 = 0; c0 < C; c0 += 512) {
        float f[8];
        load8<L>(table + (ok ? id : 0) * ldt + c0, lane, ok ? C - c0 : 0, f);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= scale;
        store8<L>(out + t * ldo + c0, lane, C - c0, f);
    }
}

// ------------------------------------------------------------------ sorting (id, position)
// A key is the id, or `vocab` for a position that takes no part (outside the table, or the padding id).
__device__ __forceinline__ int key_of(const void* ids, int wide, long long t, int vocab, long long padding) {
    const long long id = id_at(ids, wide, t);
    return id < 0 || id >= vocab || id == padding ? vocab : (int)id;
}

// Rows [row0, row1) of the table as zeros, by the workgroups of a launch behind its first `workers`.  flat: the rows are one
// range of memory, 16-byte aligned at row0.
struct Fill { float* grad; long long ldg; int C, row0, row1, workers, flat; };
__device__ __forceinline__ bool fill_part(const Fill& f) {
    if ((int)blockIdx.x < f.workers) return false;
    const long long me = (long long)(blockIdx.x - f.workers) * blockDim.x + threadIdx.x, all = (long long)(gridDim.x - f.workers) * blockDim.x;
    const long long n = (long long)(f.row1 - f.row0) * f.C;
    float* p = f.grad + f.row0 * f.ldg;
    if (f.flat) {
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        for (long long i = me; i < n / 4; i += all) __builtin_nontemporal_store(zero, (f32x4*)(p + 4 * i));  // (a table is larger than the caches: 160 -> 147 us at 131k tokens)
        if (me < (n & 3)) p[(n & ~3ll) + me] = 0.f;
    } else {  // a wave per row
        const int lane = threadIdx.x & 63;
        for (long long r = me >> 6; r < f.row1 - f.row0; r += all >> 6)
            for (int c = lane; c < f.C; c += 64) p[r * f.ldg + c] = 0.f;
    }
    return true;
}

// Up to RANK_MOST positions: one launch, every position counts the ones in front of it (T^2 comparisons of 4 bytes from LDS; with the
// zeros of half a table of 49408 x 1024 beside it, 2464 positions take 19.1 us, which is the 101 MB at 5.3 TB/s; 5003 positions alone
// 6.8 us, where the radix sort below takes four launches).  key << 13 | t orders them all, in 32 bits
// (vocab < 2^18).  A workgroup ranks 2^shift = 16 or 32 positions: 64 / 2^shift lanes of each of its 16 waves hold the same
// position and compare it with a part of all.
constexpr int RANK_MOST = 8192, RANK_VOCAB = 1 << 18;
__global__ __launch_bounds__(1024) void rank_sort_kernel(const void* ids, int wide, int T, int vocab, long long padding, int shift, int* keys, int* perm,
                                                         const Fill fill) {
    __shared__ unsigned all[RANK_MOST];
    __shared__ int part[16][32];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (fill_part(fill)) return;
    const int T4 = (T + 3) & ~3;
#pragma unroll 4
    for (int t = threadIdx.x; t < T4; t += 1024) all[t] = t < T ? (unsigned)key_of(ids, wide, t, vocab, padding) << 13 | t : 0xffffffffu;
    __syncthreads();
    const int own = 1 << shift, slices = 64 >> shift, i = lane & (own - 1), t = blockIdx.x * own + i;
    const unsigned me = all[min(t, T - 1)];
    const int quads = T4 / 4, per = (quads + 16 * slices - 1) / (16 * slices), from = (wave * slices + (lane >> shift)) * per;
    int before = 0;
#pragma unroll 8
    for (int q = from; q < min(quads, from + per); ++q) {
        const u32x4 v = *(const u32x4*)(all + 4 * q);
#pragma unroll
        for (int e = 0; e < 4; ++e) before += v[e] < me;
    }
    for (int o = own; o < 64; o <<= 1) before += __shfl_xor(before, o);
    if (lane < own) part[wave][i] = before;
    __syncthreads();
    if (wave == 0 && lane < own && t < T) {
        int r = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) r += part[w][i];
        keys[r] = (int)(me >> 13);
        perm[r] = t;
    }
}

// More positions: least significant digits first, 8 bits a pass; a workgroup takes `per` positions, in blocks of RS_BLOCK.  Every
// workgroup adds the counts hist[workgroup][digit] of the ones in front of it itself, a launch less than a scan of its own; as that
// work grows with the square of their number, there are at most RS_MOST (16.8M positions x 320: 8550 us without a limit, 3140 with
// 256, 3090 with 1024, 3075 with 512).  131071 positions and two fifths of the table's zeros each: counting 7.5 us, moving 11.7 us a
// pass, the zeros' write rate or nearly so.
constexpr int RS_BLOCK = 2048, RS_MOST = 512, RS_THREADS = 512, RS_ROUNDS = RS_BLOCK / RS_THREADS;
struct SortArgs {
    const void* ids; int wide; int T, vocab; long long padding;
    const int* keys_in; const int* perm_in;  // NULL on the first pass: the ids themselves, in order
    int* keys_out; int* perm_out;
    int* hist; int shift, per;
    Fill fill;
};
__device__ __forceinline__ int sort_key(const SortArgs& a, long long t) {
    return a.keys_in ? a.keys_in[t] : key_of(a.ids, a.wide, t, a.vocab, a.padding);
}
__global__ __launch_bounds__(RS_THREADS) void sort_hist_kernel(const SortArgs a) {
    __shared__ int h[256];
    if (fill_part(a.fill)) return;
    if (threadIdx.x < 256) h[threadIdx.x] = 0;
    __syncthreads();
    const long long t0 = (long long)blockIdx.x * a.per;
#pragma unroll 4
    for (int i = threadIdx.x; i < a.per && t0 + i < a.T; i += RS_THREADS) atomicAdd(&h[(sort_key(a, t0 + i) >> a.shift) & 255], 1);
    __syncthreads();
    if (threadIdx.x < 256) a.hist[blockIdx.x * 256 + threadIdx.x] = h[threadIdx.x];
}
__global__ __launch_bounds__(RS_THREADS) void sort_scatter_kernel(const SortArgs a) {
    constexpr int WAVES = RS_THREADS / 64;
    __shared__ int count[WAVES][256];
    __shared__ int base[2][256], total[2][256];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (fill_part(a.fill)) return;
    for (int i = tid; i < WAVES * 256; i += RS_THREADS) (&count[0][0])[i] = 0;
    // digit totals of all blocks, and of the blocks in front of this one
    {  // (half of the blocks each half of the threads)
        int before = 0, all = 0;
        const int nb = a.fill.workers, mine = blockIdx.x, half = tid >> 8, digit = tid & 255;
#pragma unroll 8
        for (int b = half; b < nb; b += 2) {
            const int v = a.hist[b * 256 + digit];
            all += v;
            before += b < mine ? v : 0;
        }
        base[half][digit] = before;
        total[half][digit] = all;
    }
    __syncthreads();
    if (wave == 0) {  // exclusive scan of the totals over the digits: 4 a lane
        int v[4], s = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) { v[e] = s; s += total[0][lane * 4 + e] + total[1][lane * 4 + e]; }
        int up = s;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int w = __shfl_up(up, o);
            if (lane >= o) up += w;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) base[0][lane * 4 + e] += base[1][lane * 4 + e] + up - s + v[e];
    }
    // a wave takes RS_ROUNDS * 64 neighbouring positions of a block in order; equal digits of a round find each other by ballots
    const long long end = min((long long)a.T, (long long)(blockIdx.x + 1) * a.per);
    for (long long block = (long long)blockIdx.x * a.per;;) {
        const long long t0 = block + wave * (RS_ROUNDS * 64);
        int key[RS_ROUNDS], perm[RS_ROUNDS], rank[RS_ROUNDS];
        volatile int* mine = count[wave];
#pragma unroll
        for (int r = 0; r < RS_ROUNDS; ++r) {
            const long long t = t0 + r * 64 + lane;
            const bool ok = t < a.T;
            key[r] = ok ? sort_key(a, t) : 0;
            perm[r] = ok ? (a.perm_in ? a.perm_in[t] : (int)t) : 0;
            const int digit = (key[r] >> a.shift) & 255;
            unsigned long long same = __ballot(ok);
#pragma unroll
            for (int b = 0; b < 8; ++b) {
                const unsigned long long has = __ballot((digit >> b) & 1);
                same &= (digit >> b) & 1 ? has : ~has;
            }
            const int lower = __popcll(same & ((1ull << lane) - 1));
            if (ok) rank[r] = mine[digit] + lower;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (ok && lower == 0) mine[digit] += __popcll(same);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
        __syncthreads();
        if (tid < 256) {  // where each wave's run of a digit begins
            int s = base[0][tid];
            for (int w = 0; w < WAVES; ++w) {
                const int c = count[w][tid];
                count[w][tid] = s;
                s += c;
            }
            base[0][tid] = s;
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < RS_ROUNDS; ++r) {
            if (t0 + r * 64 + lane < a.T) {
                const int at = count[wave][(key[r] >> a.shift) & 255] + rank[r];
                a.keys_out[at] = key[r];
                a.perm_out[at] = perm[r];
            }
        }
        block += RS_BLOCK;
        if (block >= end) return;
        __syncthreads();
        for (int i = tid; i < WAVES * 256; i += RS_THREADS) (&count[0][0])[i] = 0;
        __syncthreads();
    }
}

// ------------------------------------------------------------------ runs, and sums of whole chunks inside one
struct GradArgs {
    const int* keys; const int* perm; int T, vocab;
    const void* dy; long long lddy; int C; float scale;
    float* p64; float* p512;  // [T / 64][C], [T / 512][C]
    float* grad; long long ldg; int accumulate, per_wave;
    Fill fill;
};

// acc += rows pos[0 .. n) of dy, pos[j] in lane j (n <= 64): DEEP rows in flight, their addresses from registers
template <typename T, int L, bool PAST>
__device__ __forceinline__ void add_rows(const GradArgs& a, int pos, int n, int c0, int lane, float* acc) {
    typedef Raw<T, L, PAST> X;
    const T* dy = (const T*)a.dy + c0;
    for (int j = 0; j < n; j += X::DEEP) {
        X x[X::DEEP];
#pragma unroll
        for (int u = 0; u < X::DEEP; ++u)
            x[u].load(dy + (long long)__builtin_amdgcn_readlane(pos, min(j + u, n - 1)) * a.lddy, lane, j + u < n ? a.C - c0 : 0);
        float part[2][8] = {};  // (rows that are not there add zeros)
#pragma unroll
        for (int u = 0; u < X::DEEP; ++u) add_raw(x[u], part[u & 1]);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += part[0][e] + part[1][e];
    }
}
// acc += chunk sums first, first + 4, ... < end
template <int L>
__device__ __forceinline__ void add_chunks(const float* p, int C, int first, int end, int c0, int lane, float* acc) {
    for (int i = first; i < end; i += 16) {
        float f[4][8];
#pragma unroll
        for (int u = 0; u < 4; ++u) load8<L>(p + (long long)min(i + 4 * u, end - 1) * C + c0, lane, i + 4 * u < end ? C - c0 : 0, f[u]);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += (f[0][e] + f[1][e]) + (f[2][e] + f[3][e]);
    }
}

// Sums of 64 and of 512 sorted rows, only where they lie inside one run (the padding token of a batch of prompts): without them a
// run of thousands of rows would be one wave's chain.  Other workgroups of the launch write the last of the table's zeros (2464 rows
// of 1024 and half a table's zeros 21.8 us; 131071 rows and a fifth of the zeros 30.7 us).
// 8 waves, workgroup (b, column span): wave w sums chunk 8 b + w if it lies inside one run, together they sum chunk b of 512
template <typename T, int L, bool PAST>
__global__ __launch_bounds__(512) void chunk_sum_kernel(const GradArgs a) {
    __shared__ float red[8][512];
    __shared__ int key0[8];
    if (fill_part(a.fill)) return;
    const int spans = (a.C + 511) / 512, b = blockIdx.x / spans, c0 = (blockIdx.x - b * spans) * 512;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int s = b * 512 + wave * 64, i = s + lane;
    const int key = i < a.T ? a.keys[i] : -1, pos = i < a.T ? a.perm[i] : 0;
    const int first = __builtin_amdgcn_readfirstlane(key);
    const bool whole = first >= 0 && first < a.vocab && __all(key == first);
    float acc[8] = {};
    if (whole) {
        add_rows<T, L, PAST>(a, pos, 64, c0, lane, acc);
        store8<L>(a.p64 + (long long)(s / 64) * a.C + c0, lane, a.C - c0, acc);
    }
    if (lane == 0) key0[wave] = whole ? first : -1;
    __syncthreads();
    for (int w = 0; w < 8; ++w)
        if (key0[w] < 0 || key0[w] != key0[0]) return;  // (the same for all threads)
#pragma unroll
    for (int j = 0; j < 8; ++j) red[wave][j * 64 + lane] = acc[j];
    __syncthreads();
    if (wave == 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < 8; ++w) v += red[w][j * 64 + lane];
            acc[j] = v;
        }
        store8<L>(a.p512 + (long long)b * a.C + c0, lane, a.C - c0, acc);
    }
}

// The rows of the table that occur, each written once.  Bound by the gather of dy's rows outside whole chunks: 131071 rows of 1024 bf16
// 62.9 us (with the chunks' sums 94 us for 268 MB read, the occurring rows and the last zeros written); 2464 rows 7.1 us.
// grid (T / 4 per_wave rounded up, C / 512 rounded up), 4 waves: a wave takes the runs that begin in its per_wave <= 32 sorted
// positions.  Runs of up to 32 positions it streams one after the other, eight positions at a time, across their borders.  A longer
// one (at most one begins there, the last) is summed by the four waves together, from the chunk sums where they cover it.
constexpr int RUN_SHORT = 32;
template <typename T, int L, bool PAST>
__global__ __launch_bounds__(256) void run_sum_kernel(const GradArgs a) {
    __shared__ float red[4][512];
    __shared__ int long_at[4];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c0 = blockIdx.y * 512, cols = a.C - c0;
    auto put = [&](long long v, float* acc) {
        float* row = a.grad + v * a.ldg + c0;
        if (a.accumulate) {
            float old[8];
            load8<L>(row, lane, cols, old);
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] = fmaf(acc[j], a.scale, old[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] *= a.scale;
        }
        store8<L>(row, lane, cols, acc);
    };
    // this wave's positions and the 32 behind them: where runs begin (a position behind the last counts as a beginning)
    const int p0 = (blockIdx.x * 4 + wave) * a.per_wave, p = p0 + lane;
    const int key = p < a.T ? a.keys[p] : a.vocab, pos = p < a.T ? a.perm[p] : 0;
    const int front = p0 > 0 && p0 < a.T ? a.keys[p0 - 1] : -1, up = __shfl_up(key, 1);
    const bool begins = p >= a.T || key != (lane == 0 ? front : up);
    const unsigned long long marks = __ballot(begins), live = __ballot(key < a.vocab);  // (live positions come first)
    const unsigned mine = (unsigned)marks & (unsigned)live & (0xffffffffu >> (32 - a.per_wave));
    int begin = 0, end = 0, long_s = -1;
    if (mine) {
        begin = __ffs(mine) - 1;
        const int last = 31 - __clz(mine);  // the last run that begins here
        const unsigned long long behind = marks >> last >> 1;
        const int len = behind ? __ffsll(behind) : 64;
        if (len > RUN_SHORT) long_s = p0 + last;
        end = len > RUN_SHORT ? last : last + len;
    }
    const T* dy = (const T*)a.dy + c0;
    {
        float acc[8] = {};
        int row = -1;
        for (int j = begin; j < end; j += 8) {
            Raw<T, L, PAST> x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u)
                x[u].load(dy + (long long)__builtin_amdgcn_readlane(pos, min(j + u, end - 1)) * a.lddy, lane, j + u < end ? cols : 0);
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (j + u < end) {
                    const int k = __builtin_amdgcn_readlane(key, j + u);
                    if (k != row) {
                        if (row >= 0) put(row, acc);
                        row = k;
#pragma unroll
                        for (int e = 0; e < 8; ++e) acc[e] = 0.f;
                    }
                    add_raw(x[u], acc);
                }
        }
        if (row >= 0) put(row, acc);
    }
    if (lane == 0) long_at[wave] = long_s;
    __syncthreads();
    for (int w = 0; w < 4; ++w) {
        const int s = __builtin_amdgcn_readfirstlane(long_at[w]);
        if (s < 0) continue;
        const int v = a.keys[s];
        int lo = s + RUN_SHORT, e = a.T;  // keys[lo] is the run's, position e is not: 64 probes a round
        while (e - lo > 1) {
            const int n = e - lo, at = lo + (int)((long long)n * (lane + 1) / 65);
            const int in = __popcll(__ballot(a.keys[at] == v));
            const int l2 = in == 0 ? lo : lo + (int)((long long)n * in / 65), e2 = in == 64 ? e : lo + (int)((long long)n * (in + 1) / 65);
            if (l2 == lo && e2 == e) break;  // (not reached: a round cuts n to at most n / 65 + 1)
            lo = l2;
            e = e2;
        }
        // rows [s, 64 ca), chunks [ca, 8 da) of 64, chunks [da, db) of 512, chunks [8 db, cb) of 64, rows [64 cb, e)
        float acc[8] = {};
        const int ca = (s + 63) / 64, cb = e / 64, da = (ca + 7) / 8, db = cb / 8;
        auto rows = [&](int from, int to) {  // at most 126: every fourth of them a wave's
            const int cnt = (to - from - wave + 3) / 4;
            if (cnt <= 0) return;
            const int at = lane < cnt ? a.perm[from + wave + 4 * lane] : 0;
            add_rows<T, L, PAST>(a, at, cnt, c0, lane, acc);
        };
        if (ca >= cb) {
            rows(s, e);
        } else {
            rows(s, ca * 64);
            if (da >= db) {
                add_chunks<L>(a.p64, a.C, ca + wave, cb, c0, lane, acc);
            } else {
                add_chunks<L>(a.p64, a.C, ca + wave, da * 8, c0, lane, acc);
                add_chunks<L>(a.p512, a.C, da + wave, db, c0, lane, acc);
                add_chunks<L>(a.p64, a.C, db * 8 + wave, cb, c0, lane, acc);
            }
            rows(cb * 64, e);
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) red[wave][j * 64 + lane] = acc[j];
        __syncthreads();
        if (wave == 0) {
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] = (red[0][j * 64 + lane] + red[1][j * 64 + lane]) + (red[2][j * 64 + lane] + red[3][j * 64 + lane]);
            put(v, acc);
        }
    }
}

template <typename TW, typename TO>
void launch_lookup(bool vec, const void* ids, int wide, int T, int vocab, const void* table, int ldt, int C, float scale, void* out, int ldo,
                   hipStream_t st) {
    constexpr int OTHER = sizeof(TW) == 4 && sizeof(TO) == 4 ? SPREAD : LOOSE;
    constexpr int MOST = 1 << 25;  // (a launch has less than 2^32 threads)
    for (long long t = 0; t < T; t += MOST) {
        const int n = (int)std::min<long long>(T - t, MOST);
        const dim3 grid((unsigned)((n + 3) / 4));
        const void* id = (const char*)ids + t * (wide ? 8 : 4);
        TO* to = (TO*)out + t * ldo;
        if (vec) hipLaunchKernelGGL((lookup_kernel<TW, TO, VECTOR>), grid, dim3(256), 0, st, id, wide, n, vocab, (const TW*)table, (long long)ldt, C, scale, to, (long long)ldo);
        else hipLaunchKernelGGL((lookup_kernel<TW, TO, OTHER>), grid, dim3(256), 0, st, id, wide, n, vocab, (const TW*)table, (long long)ldt, C, scale, to, (long long)ldo);
    }
}

template <typename T, int L, bool PAST>
int launch_grad(GradArgs a, unsigned fillers, hipStream_t st) {
    // few positions a wave while the grid is small (2464 positions: 41 us against 46 with 16), more where waves abound (131071: 145 / 147)
    a.per_wave = a.T <= 65536 ? 8 : 16;
    const unsigned spans = (unsigned)((a.C + 511) / 512);
    hipLaunchKernelGGL((chunk_sum_kernel<T, L, PAST>), dim3((unsigned)a.fill.workers + fillers), dim3(512), 0, st, a);
    CCNET_LAUNCH_CHECK();
    hipLaunchKernelGGL((run_sum_kernel<T, L, PAST>), dim3((unsigned)((a.T + 4 * a.per_wave - 1) / (4 * a.per_wave)), spans), dim3(256), 0, st, a);
    CCNET_LAUNCH_CHECK();
    return CCNET_OK;
}

bool aligned16(const void* p, long long ld, int esz) { return !((uintptr_t)p & 15) && (ld * esz) % 16 == 0; }

int sort_per(int T) { return T > 0 ? ((T - 1) / (RS_MOST * RS_BLOCK) + 1) * RS_BLOCK : RS_BLOCK; }

// workspace: sorted keys and positions (twice: a pass reads one copy and writes the other), digit counts, chunk sums
struct Layout { size_t keys[2], perm[2], hist, p64, p512, bytes; };
Layout layout_of(int T, int C) {
    Layout l{};
    size_t at = 0;
    auto take = [&](size_t n) { const size_t r = at; at += (n + 255) & ~(size_t)255; return r; };
    for (int i = 0; i < 2; ++i) { l.keys[i] = take((size_t)T * 4); l.perm[i] = take((size_t)T * 4); }
    l.hist = take(((size_t)T + sort_per(T) - 1) / sort_per(T) * 1024);
    l.p64 = take((size_t)(T / 64) * C * 4);
    l.p512 = take((size_t)(T / 512) * C * 4);
    l.bytes = at;
    return l;
}

}  // namespace

extern "C" int ccnet_embedding(const void* ids, int id_bytes, int T, int vocab, const void* table, int table_dtype, int ldt, int C,
                               float scale, void* out, int out_dtype, int ldo, void* stream) {
    if (T < 0 || vocab <= 0 || C <= 0 || (id_bytes != 4 && id_bytes != 8) || table_dtype < 0 || table_dtype > 1 || out_dtype < 0 || out_dtype > 1 ||
        ldt < C || ldo < C)
        return CCNET_EINVAL;
    if (T == 0) return CCNET_OK;
    const int ws = table_dtype == 0 ? 4 : 2, os = out_dtype == 0 ? 4 : 2;
    if (!ids || !table || !out || (uintptr_t)ids % id_bytes || (uintptr_t)table % ws || (uintptr_t)out % os) return CCNET_EINVAL;
    const RowSpan to{out, (long long)ldo * os, (long long)C * os, T};
    if (!spans_apart(to, {table, (long long)ldt * ws, (long long)C * ws, vocab}) || !spans_apart(to, {ids, id_bytes, id_bytes, T})) return CCNET_EINVAL;
    const bool vec = C % 8 == 0 && aligned16(table, ldt, ws) && aligned16(out, ldo, os);
    hipStream_t st = (hipStream_t)stream;
    const int wide = id_bytes == 8;
    if (table_dtype == 0 && out_dtype == 0) launch_lookup<float, float>(vec, ids, wide, T, vocab, table, ldt, C, scale, out, ldo, st);
    else if (table_dtype == 0) launch_lookup<float, bf16_t>(vec, ids, wide, T, vocab, table, ldt, C, scale, out, ldo, st);
    else if (out_dtype == 0) launch_lookup<bf16_t, float>(vec, ids, wide, T, vocab, table, ldt, C, scale, out, ldo, st);
    else launch_lookup<bf16_t, bf16_t>(vec, ids, wide, T, vocab, table, ldt, C, scale, out, ldo, st);
    CCNET_LAUNCH_CHECK();
    return CCNET_OK;
}

extern "C" size_t ccnet_embedding_grad_workspace_bytes(int T, int C) {
    if (T <= 0 || C <= 0) return 0;
    return layout_of(T, C).bytes;
}

extern "C" int ccnet_embedding_grad(const void* ids, int id_bytes, int T, int vocab, const void* dy, int dy_dtype, int lddy, int C,
                                    float scale, int64_t padding_idx, float* grad, int ldg, int accumulate, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    if (T < 0 || vocab <= 0 || vocab == 0x7fffffff || C <= 0 || (id_bytes != 4 && id_bytes != 8) || dy_dtype < 0 || dy_dtype > 1 || lddy < C || ldg < C)
        return CCNET_EINVAL;
    if (T > (1 << 29) || ((long long)T / 512 + 1) * ((C + 511) / 512) > 0x3fffffffLL) return CCNET_EUNSUP;
    const int ds = dy_dtype == 0 ? 4 : 2;
    if (!grad || ((uintptr_t)grad & 3) || (C + 511) / 512 > 65535) return CCNET_EINVAL;
    if (T > 0 && (!ids || !dy || (uintptr_t)ids % id_bytes || (uintptr_t)dy % ds)) return CCNET_EINVAL;
    const Layout l = layout_of(T, C);
    if (T > 0 && (!workspace || ((uintptr_t)workspace & 15))) return CCNET_EINVAL;
    if (T > 0 && workspace_bytes < l.bytes) return CCNET_EWS;
    const RowSpan to{grad, (long long)ldg * 4, (long long)C * 4, vocab};
    if (!spans_apart(to, {dy, (long long)lddy * ds, (long long)C * ds, T}) || !spans_apart(to, {ids, id_bytes, id_bytes, T})) return CCNET_EINVAL;
    const RowSpan used{workspace, (long long)l.bytes, (long long)l.bytes, T > 0};
    if (!spans_apart(used, to) || !spans_apart(used, {dy, (long long)lddy * ds, (long long)C * ds, T}) || !spans_apart(used, {ids, id_bytes, id_bytes, T}))
        return CCNET_EINVAL;
    if (T == 0 && accumulate) return CCNET_OK;
    hipStream_t st = (hipStream_t)stream;
    // the table's zeros in parts [0, vocab): part k of n with a launch that has `workers` workgroups of its own
    const bool flat = ldg == C && !((uintptr_t)grad & 15);
    int filled = 0;
    unsigned fillers = 0;
    auto fill_next = [&](int workers, int k, int n) {
        Fill f{grad, ldg, C, filled, accumulate ? filled : k == n ? vocab : (int)((long long)vocab * k / n / 4 * 4), workers, flat};
        filled = f.row1;
        const long long bytes = (long long)(f.row1 - f.row0) * C * 4;  // 32 KiB a workgroup, at most 8 a CU
        fillers = bytes <= 0 ? 0u : (unsigned)std::min<long long>((bytes + 32767) / 32768, 2048);
        return f;
    };
    if (T == 0) {
        SortArgs s{};
        s.fill = fill_next(0, 1, 1);
        hipLaunchKernelGGL(sort_hist_kernel, dim3(fillers), dim3(RS_THREADS), 0, st, s);
        CCNET_LAUNCH_CHECK();
        return CCNET_OK;
    }
    char* ws = (char*)workspace;
    GradArgs g{};
    g.T = T; g.vocab = vocab; g.dy = dy; g.lddy = lddy; g.C = C; g.scale = scale; g.grad = grad; g.ldg = ldg; g.accumulate = accumulate != 0;
    g.p64 = (float*)(ws + l.p64);
    g.p512 = (float*)(ws + l.p512);
    int* keys[2] = {(int*)(ws + l.keys[0]), (int*)(ws + l.keys[1])};
    int* perm[2] = {(int*)(ws + l.perm[0]), (int*)(ws + l.perm[1])};
    int cur = 0, passes = 0;
    const int chunk_workers = (int)((T + 511) / 512) * ((C + 511) / 512);
    if (T <= RANK_MOST && vocab < RANK_VOCAB) {
        const int shift = T <= 4096 ? 4 : 5;  // (at most 256 workgroups: one a CU)
        const Fill f = fill_next((T + (1 << shift) - 1) >> shift, 1, 2);
        hipLaunchKernelGGL(rank_sort_kernel, dim3(f.workers + fillers), dim3(1024), 0, st, ids, (int)(id_bytes == 8), T, vocab, (long long)padding_idx, shift,
                           keys[0], perm[0], f);
        CCNET_LAUNCH_CHECK();
        passes = 1;
    } else {
        SortArgs s{};
        s.ids = ids; s.wide = id_bytes == 8; s.T = T; s.vocab = vocab; s.padding = padding_idx; s.hist = (int*)(ws + l.hist);
        s.per = sort_per(T);
        const int blocks = (T - 1) / s.per + 1;
        for (int shift = 0; shift < 32 && (vocab >> shift) > 0; shift += 8) passes += 2;
        cur = 1;
        for (int k = 0; k < passes; k += 2) {
            s.shift = 4 * k;
            s.keys_out = keys[1 - cur]; s.perm_out = perm[1 - cur];
            s.fill = fill_next(blocks, k + 1, passes + 1);
            hipLaunchKernelGGL(sort_hist_kernel, dim3(blocks + fillers), dim3(RS_THREADS), 0, st, s);
            CCNET_LAUNCH_CHECK();
            s.fill = fill_next(blocks, k + 2, passes + 1);
            hipLaunchKernelGGL(sort_scatter_kernel, dim3(blocks + fillers), dim3(RS_THREADS), 0, st, s);
            CCNET_LAUNCH_CHECK();
            cur = 1 - cur;
            s.keys_in = keys[cur]; s.perm_in = perm[cur];
        }
    }
    g.keys = keys[cur];
    g.perm = perm[cur];
    g.fill = fill_next(chunk_workers, passes + 1, passes + 1);
    const bool vec = C % 8 == 0 && aligned16(dy, lddy, ds) && aligned16(grad, ldg, 4);
    const bool past = (long long)T * C * ds > 192ll << 20;  // (the memory-side cache holds 256 MiB)
    auto go = [&](auto zero) {
        typedef decltype(zero) D;
        constexpr int OTHER = sizeof(D) == 4 ? SPREAD : LOOSE;
        if (vec) return past ? launch_grad<D, VECTOR, true>(g, fillers, st) : launch_grad<D, VECTOR, false>(g, fillers, st);
        return past && OTHER == LOOSE ? launch_grad<D, OTHER, OTHER == LOOSE>(g, fillers, st) : launch_grad<D, OTHER, false>(g, fillers, st);
    };
    return dy_dtype == 0 ? go(float{}) : go(bf16_t{});
}
