// Token lookup with scaling, and its gradient by sorted tokens.
//
//   y[t] = scale * W[id[t]]                      (ids outside [0, vocab): a row of zeros)
//   dW[v] = scale * sum over t with id[t] = v of dy[t], in rising t
//
// The gradient sorts (id, t) and then writes every row of dW once, in fp32, from a fixed tree over the row's run of sorted
// positions: no float atomics, so equal inputs give equal bits.  A run may hold one position or nearly all of them (the
// padding token of a batch of prompts), so runs are summed in three grains: single rows, whole aligned chunks of 64
// sorted positions and whole aligned chunks of 512 that lie inside one run (run_kernel), joined by
// table_grad_kernel.  Rows without a token are written as zeros by the same kernel.
#include "common.h"

namespace {

typedef unsigned short bf16_t;
typedef __attribute__((ext_vector_type(2))) int i32x2;

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(bf16_t v) { return bf16_bits_to_f32(v); }
__device__ __forceinline__ void from_f32(float& d, float v) { d = v; }
__device__ __forceinline__ void from_f32(bf16_t& d, float v) { d = f32_to_bf16_bits(v); }

// Eight columns of a 512-column span a lane: VEC 8 neighbours (16-byte accesses), else every 64th.
template <bool VEC>
__device__ __forceinline__ int col_of(int lane, int j) { return VEC ? lane * 8 + j : lane + 64 * j; }
template <bool VEC>
__device__ __forceinline__ void load8(const float* row, int lane, int cols, float* f) {
    if constexpr (VEC) {
        f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
        if (lane * 8 < cols) {
            a = *(const f32x4*)(row + lane * 8);
            b = *(const f32x4*)(row + lane * 8 + 4);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) { f[e] = a[e]; f[4 + e] = b[e]; }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = lane + 64 * j < cols ? row[lane + 64 * j] : 0.f;
    }
}
template <bool VEC>
__device__ __forceinline__ void load8(const bf16_t* row, int lane, int cols, float* f) {
    if constexpr (VEC) {
        u32x4 a = {0u, 0u, 0u, 0u};
        if (lane * 8 < cols) a = *(const u32x4*)(row + lane * 8);
        unpack8(a, f);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = lane + 64 * j < cols ? bf16_bits_to_f32(row[lane + 64 * j]) : 0.f;
    }
}
template <bool VEC>
__device__ __forceinline__ void store8(float* row, int lane, int cols, const float* f) {
    if constexpr (VEC) {
        if (lane * 8 < cols) {
            *(f32x4*)(row + lane * 8) = f32x4{f[0], f[1], f[2], f[3]};
            *(f32x4*)(row + lane * 8 + 4) = f32x4{f[4], f[5], f[6], f[7]};
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (lane + 64 * j < cols) row[lane + 64 * j] = f[j];
    }
}
template <bool VEC>
__device__ __forceinline__ void store8(bf16_t* row, int lane, int cols, const float* f) {
    if constexpr (VEC) {
        if (lane * 8 < cols) *(u32x4*)(row + lane * 8) = pack8(f);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (lane + 64 * j < cols) row[lane + 64 * j] = f32_to_bf16_bits(f[j]);
    }
}

__device__ __forceinline__ long long id_at(const void* ids, int wide, long long t) {
    return wide ? ((const long long*)ids)[t] : (long long)((const int*)ids)[t];
}

// ------------------------------------------------------------------ lookup: a wave per row and 512 columns
template <typename TW, typename TO, bool VEC>
__global__ __launch_bounds__(256) void lookup_kernel(const void* ids, int wide, int T, int vocab, const TW* table, long long ldt, int C,
                                                     float scale, TO* out, long long ldo) {
    const int lane = threadIdx.x & 63;
    const long long t = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= T) return;
    const long long id = id_at(ids, wide, t);
    const bool ok = id >= 0 && id < vocab;
    for (int c0 = 0; c0 < C; c0 += 512) {
        float f[8];
        load8<VEC>(table + (ok ? id : 0) * ldt + c0, lane, ok ? C - c0 : 0, f);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= scale;
        store8<VEC>(out + t * ldo + c0, lane, C - c0, f);
    }
}

// ------------------------------------------------------------------ sorting (id, position)
// A key is the id, or `vocab` for a position that takes no part (outside the table, or the padding id).
__device__ __forceinline__ int key_of(const void* ids, int wide, long long t, int vocab, long long padding) {
    const long long id = id_at(ids, wide, t);
    return id < 0 || id >= vocab || id == padding ? vocab : (int)id;
}

// every id's run of sorted positions [first, end): none yet
__device__ __forceinline__ void clear_runs(i32x2* runs, int vocab) {
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < vocab; i += (long long)gridDim.x * blockDim.x) runs[i] = i32x2{0, 0};
}

// Up to RANK_MOST positions: every position counts the ones in front of it.  key << 13 | t orders them all, in 32 bits
// (vocab < 2^18); 64 positions a workgroup, its 16 waves each compare them with a sixteenth of all.
constexpr int RANK_MOST = 8192, RANK_VOCAB = 1 << 18;
__global__ __launch_bounds__(1024) void rank_sort_kernel(const void* ids, int wide, int T, int vocab, long long padding, int* keys, int* perm, i32x2* runs) {
    __shared__ unsigned all[RANK_MOST];
    __shared__ int part[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    clear_runs(runs, vocab);
    if ((int)blockIdx.x * 64 >= T) return;
    const int T4 = (T + 3) & ~3;
    for (int t = threadIdx.x; t < T4; t += 1024) all[t] = t < T ? (unsigned)key_of(ids, wide, t, vocab, padding) << 13 | t : 0xffffffffu;
    __syncthreads();
    const int t = blockIdx.x * 64 + lane;
    const unsigned me = all[min(t, T - 1)];
    const int quads = T4 / 4, per = (quads + 15) / 16;
    int before = 0;
#pragma unroll 8
    for (int i = wave * per; i < min(quads, (wave + 1) * per); ++i) {
        const u32x4 v = *(const u32x4*)(all + 4 * i);
#pragma unroll
        for (int e = 0; e < 4; ++e) before += v[e] < me;
    }
    part[wave][lane] = before;
    __syncthreads();
    if (wave == 0 && t < T) {
        int r = 0;
        for (int w = 0; w < 16; ++w) r += part[w][lane];
        keys[r] = (int)(me >> 13);
        perm[r] = t;
    }
}

// More positions: least significant digits first, 8 bits a pass, RS_BLOCK positions a workgroup.  hist[block][digit].
constexpr int RS_BLOCK = 2048, RS_THREADS = 512, RS_ROUNDS = RS_BLOCK / RS_THREADS;
struct SortArgs {
    const void* ids; int wide; int T, vocab; long long padding;
    const int* keys_in; const int* perm_in;  // NULL on the first pass: the ids themselves, in order
    int* keys_out; int* perm_out;
    int* hist; int shift;
    i32x2* runs;  // cleared on the first pass
};
__device__ __forceinline__ int sort_key(const SortArgs& a, long long t) {
    return a.keys_in ? a.keys_in[t] : key_of(a.ids, a.wide, t, a.vocab, a.padding);
}
__global__ __launch_bounds__(RS_THREADS) void sort_hist_kernel(const SortArgs a) {
    __shared__ int h[256];
    if (threadIdx.x < 256) h[threadIdx.x] = 0;
    if (a.shift == 0) clear_runs(a.runs, a.vocab);
    __syncthreads();
    const long long t0 = (long long)blockIdx.x * RS_BLOCK;
    for (int i = threadIdx.x; i < RS_BLOCK && t0 + i < a.T; i += RS_THREADS) atomicAdd(&h[(sort_key(a, t0 + i) >> a.shift) & 255], 1);
    __syncthreads();
    if (threadIdx.x < 256) a.hist[blockIdx.x * 256 + threadIdx.x] = h[threadIdx.x];
}
__global__ __launch_bounds__(RS_THREADS) void sort_scatter_kernel(const SortArgs a) {
    constexpr int WAVES = RS_THREADS / 64;
    __shared__ int count[WAVES][256];
    __shared__ int base[2][256], total[2][256];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int i = tid; i < WAVES * 256; i += RS_THREADS) (&count[0][0])[i] = 0;
    // digit totals of all blocks, and of the blocks in front of this one
    {  // (half of the blocks each half of the threads)
        int before = 0, all = 0;
        const int nb = gridDim.x, mine = blockIdx.x, half = tid >> 8, digit = tid & 255;
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
    // a wave takes RS_ROUNDS * 64 neighbouring positions in order; equal digits of a round find each other by ballots
    const long long t0 = (long long)blockIdx.x * RS_BLOCK + wave * (RS_ROUNDS * 64);
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
}

// ------------------------------------------------------------------ runs, and sums of whole chunks inside one
struct GradArgs {
    const int* keys; const int* perm; int T, vocab;
    const void* dy; long long lddy; int C; float scale;
    i32x2* runs;              // [vocab]
    float* p64; float* p512;  // [T / 64][C], [T / 512][C]
    float* grad; long long ldg; int accumulate, rows_per_wave;
};

// Eight columns as they lie in memory, so that many rows in flight cost no more registers than their bytes.
template <typename T, bool VEC> struct Raw;
template <> struct Raw<float, true> {
    static constexpr int DEEP = 8;
    f32x4 a, b;
    __device__ __forceinline__ void load(const float* row, int lane, int cols) {
        a = b = f32x4{0.f, 0.f, 0.f, 0.f};
        if (lane * 8 < cols) { a = *(const f32x4*)(row + lane * 8); b = *(const f32x4*)(row + lane * 8 + 4); }
    }
    __device__ __forceinline__ void add(float* acc) const {
#pragma unroll
        for (int e = 0; e < 4; ++e) { acc[e] += a[e]; acc[4 + e] += b[e]; }
    }
};
template <> struct Raw<bf16_t, true> {
    static constexpr int DEEP = 16;
    u32x4 a;
    __device__ __forceinline__ void load(const bf16_t* row, int lane, int cols) {
        a = u32x4{0u, 0u, 0u, 0u};
        if (lane * 8 < cols) a = *(const u32x4*)(row + lane * 8);
    }
    __device__ __forceinline__ void add(float* acc) const {
        float f[8];
        unpack8(a, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += f[e];
    }
};
template <typename T> struct Raw<T, false> {
    static constexpr int DEEP = 8;
    T v[8];
    __device__ __forceinline__ void load(const T* row, int lane, int cols) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = lane + 64 * j < cols ? row[lane + 64 * j] : (T)0;
    }
    __device__ __forceinline__ void add(float* acc) const {
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += to_f32(v[j]);
    }
};

// acc += rows pos[0 .. n) of dy, pos[j] in lane j (n <= 64): DEEP rows in flight, their addresses from registers
template <typename T, bool VEC>
__device__ __forceinline__ void add_rows(const GradArgs& a, int pos, int n, int c0, int lane, float* acc) {
    typedef Raw<T, VEC> X;
    const T* dy = (const T*)a.dy + c0;
    for (int j = 0; j < n; j += X::DEEP) {
        X x[X::DEEP];
#pragma unroll
        for (int u = 0; u < X::DEEP; ++u)
            x[u].load(dy + (long long)__builtin_amdgcn_readlane(pos, min(j + u, n - 1)) * a.lddy, lane, j + u < n ? a.C - c0 : 0);
        float part[2][8] = {};  // (rows that are not there add zeros)
#pragma unroll
        for (int u = 0; u < X::DEEP; ++u) x[u].add(part[u & 1]);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += part[0][e] + part[1][e];
    }
}
// acc += chunk sums first, first + 4, ... < end
template <bool VEC>
__device__ __forceinline__ void add_chunks(const float* p, int C, int first, int end, int c0, int lane, float* acc) {
    for (int i = first; i < end; i += 16) {
        float f[4][8];
#pragma unroll
        for (int u = 0; u < 4; ++u) load8<VEC>(p + (long long)min(i + 4 * u, end - 1) * C + c0, lane, i + 4 * u < end ? C - c0 : 0, f[u]);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] += (f[0][e] + f[1][e]) + (f[2][e] + f[3][e]);
    }
}

// grid (T / 512 rounded up, C / 512 rounded up), 8 waves: wave w marks where runs begin and end in chunk 8 b + w, and sums the
// chunk if it lies inside one run
template <typename T, bool VEC>
__global__ __launch_bounds__(512) void run_kernel(const GradArgs a) {
    __shared__ float red[8][512];
    __shared__ int key0[8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c0 = blockIdx.y * 512;
    const int s = blockIdx.x * 512 + wave * 64, i = s + lane;
    const int key = i < a.T ? a.keys[i] : -1, prev = i > 0 && i < a.T ? a.keys[i - 1] : -1;
    const int pos = i < a.T ? a.perm[i] : 0;
    if (blockIdx.y == 0 && i < a.T) {
        if (key != prev) {
            if (key < a.vocab) ((int*)a.runs)[2ll * key] = i;
            if (prev >= 0) ((int*)a.runs)[2ll * prev + 1] = i;  // (the positions that take no part sort last: prev < vocab)
        }
        if (i == a.T - 1 && key < a.vocab) ((int*)a.runs)[2ll * key + 1] = a.T;
    }
    const int first = __builtin_amdgcn_readfirstlane(key);
    const bool whole = first >= 0 && first < a.vocab && __all(key == first);
    float acc[8] = {};
    if (whole) {
        add_rows<T, VEC>(a, pos, 64, c0, lane, acc);
        store8<VEC>(a.p64 + (long long)(s / 64) * a.C + c0, lane, a.C - c0, acc);
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
        store8<VEC>(a.p512 + (long long)blockIdx.x * a.C + c0, lane, a.C - c0, acc);
    }
}

// grid (G, C / 512 rounded up), 4 waves of R = rows_per_wave <= TG_ROWS rows.  A wave writes R neighbouring rows whose runs are
// short: their sorted positions are neighbours too, so it streams them eight at a time across the rows' borders.  Long runs are
// summed by the four waves together; those of the workgroup are rows blockIdx.x + i G, as frequent ids are neighbours in a
// vocabulary.
constexpr int TG_ROWS = 4, TG_SHORT = 32;
template <typename T, bool VEC>
__global__ __launch_bounds__(256) void table_grad_kernel(const GradArgs a) {
    __shared__ float red[4][512];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), c0 = blockIdx.y * 512, cols = a.C - c0;
    const int R = a.rows_per_wave;
    const long long v0 = (long long)blockIdx.x * 4 * R + wave * R;
    i32x2 mine = {0, 0}, strided = {0, 0};
    if (a.T > 0 && lane < R && v0 + lane < a.vocab) mine = a.runs[v0 + lane];
    const long long vs = blockIdx.x + (long long)lane * gridDim.x;
    if (a.T > 0 && lane < 4 * R && vs < a.vocab) strided = a.runs[vs];
    auto put = [&](long long v, float* acc) {
        float* row = a.grad + v * a.ldg + c0;
        if (a.accumulate) {
            float old[8];
            load8<VEC>(row, lane, cols, old);
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] = fmaf(acc[j], a.scale, old[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] *= a.scale;
        }
        store8<VEC>(row, lane, cols, acc);
    };
    const int n = mine[1] - mine[0];
    if (!a.accumulate) {
        for (int r = 0; r < R; ++r)
            if (v0 + r < a.vocab && __builtin_amdgcn_readlane(n, r) == 0) {
                const float zero[8] = {};
                store8<VEC>(a.grad + (v0 + r) * a.ldg + c0, lane, cols, zero);
            }
    }
    // short runs: from row to row while their positions follow each other
    const T* dy = (const T*)a.dy + c0;
    for (int r = 0; r < R;) {
        const int begin = __builtin_amdgcn_readlane(mine[0], r);
        int end = begin, r1 = r;
        for (; r1 < R; ++r1) {
            const int k = __builtin_amdgcn_readlane(n, r1);
            if (k > TG_SHORT) break;
            if (k == 0) {
                if (end == begin) break;  // (nothing yet: the next row starts anew)
                continue;
            }
            end = __builtin_amdgcn_readlane(mine[1], r1);
        }
        float acc[8] = {};
        long long row = -1;
        for (int p0 = begin; p0 < end; p0 += 64) {
            const int left = min(end - p0, 64);
            const int key = lane < left ? a.keys[p0 + lane] : 0, pos = lane < left ? a.perm[p0 + lane] : 0;
            for (int j = 0; j < left; j += 8) {
                Raw<T, VEC> x[8];
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    x[u].load(dy + (long long)__builtin_amdgcn_readlane(pos, min(j + u, left - 1)) * a.lddy, lane, j + u < left ? cols : 0);
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    if (j + u < left) {
                        const int k = __builtin_amdgcn_readlane(key, j + u);
                        if (k != row) {
                            if (row >= 0) put(row, acc);
                            row = k;
#pragma unroll
                            for (int e = 0; e < 8; ++e) acc[e] = 0.f;
                        }
                        x[u].add(acc);
                    }
            }
        }
        if (row >= 0) put(row, acc);
        r = r1 > r ? r1 : r + 1;
    }
    // long runs
    unsigned long long todo = __ballot(strided[1] - strided[0] > TG_SHORT);
    while (todo) {
        const int i = __ffsll((unsigned long long)todo) - 1;
        todo &= todo - 1;
        const int s = __builtin_amdgcn_readlane(strided[0], i), e = __builtin_amdgcn_readlane(strided[1], i);
        const long long v = blockIdx.x + (long long)i * gridDim.x;
        // rows [s, 64 ca), chunks [ca, 8 da) of 64, chunks [da, db) of 512, chunks [8 db, cb) of 64, rows [64 cb, e)
        float acc[8] = {};
        const int ca = (s + 63) / 64, cb = e / 64, da = (ca + 7) / 8, db = cb / 8;
        auto rows = [&](int from, int to) {  // at most 192: every fourth of them a wave's
            const int cnt = (to - from - wave + 3) / 4;
            if (cnt <= 0) return;
            const int pos = lane < cnt ? a.perm[from + wave + 4 * lane] : 0;
            add_rows<T, VEC>(a, pos, cnt, c0, lane, acc);
        };
        if (ca >= cb) {
            rows(s, e);
        } else {
            rows(s, ca * 64);
            if (da >= db) {
                add_chunks<VEC>(a.p64, a.C, ca + wave, cb, c0, lane, acc);
            } else {
                add_chunks<VEC>(a.p64, a.C, ca + wave, da * 8, c0, lane, acc);
                add_chunks<VEC>(a.p512, a.C, da + wave, db, c0, lane, acc);
                add_chunks<VEC>(a.p64, a.C, db * 8 + wave, cb, c0, lane, acc);
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
    const dim3 grid((unsigned)(((long long)T + 3) / 4));
    if (vec) hipLaunchKernelGGL((lookup_kernel<TW, TO, true>), grid, dim3(256), 0, st, ids, wide, T, vocab, (const TW*)table, (long long)ldt, C, scale, (TO*)out, (long long)ldo);
    else hipLaunchKernelGGL((lookup_kernel<TW, TO, false>), grid, dim3(256), 0, st, ids, wide, T, vocab, (const TW*)table, (long long)ldt, C, scale, (TO*)out, (long long)ldo);
}

template <typename T, bool VEC>
int launch_grad(GradArgs a, hipStream_t st) {
    const unsigned ct = (unsigned)((a.C + 511) / 512);
    if (a.T > 0) {
        hipLaunchKernelGGL((run_kernel<T, VEC>), dim3((unsigned)(((long long)a.T + 511) / 512), ct), dim3(512), 0, st, a);
        CCNET_LAUNCH_CHECK();
    }
    // four rows a wave where that still fills the chip (256 CUs x 8 workgroups of four waves), one in smaller tables
    a.rows_per_wave = a.vocab >= 16 * 1024 ? TG_ROWS : 1;
    const long long per = 4ll * a.rows_per_wave;
    hipLaunchKernelGGL((table_grad_kernel<T, VEC>), dim3((unsigned)((a.vocab + per - 1) / per), ct), dim3(256), 0, st, a);
    CCNET_LAUNCH_CHECK();
    return CCNET_OK;
}

bool aligned16(const void* p, long long ld, int esz) { return !((uintptr_t)p & 15) && (ld * esz) % 16 == 0; }

// workspace: sorted keys and positions (twice: a pass reads one copy and writes the other), digit counts, chunk sums
struct Layout { size_t keys[2], perm[2], hist, runs, p64, p512, bytes; };
Layout layout_of(int T, int vocab, int C) {
    Layout l{};
    size_t at = 0;
    auto take = [&](size_t n) { const size_t r = at; at += (n + 255) & ~(size_t)255; return r; };
    for (int i = 0; i < 2; ++i) { l.keys[i] = take((size_t)T * 4); l.perm[i] = take((size_t)T * 4); }
    l.hist = take(((size_t)T + RS_BLOCK - 1) / RS_BLOCK * 1024);
    l.runs = take((size_t)vocab * 8);
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

extern "C" size_t ccnet_embedding_grad_workspace_bytes(int T, int vocab, int C) {
    if (T <= 0 || vocab <= 0 || C <= 0) return 0;
    return layout_of(T, vocab, C).bytes;
}

extern "C" int ccnet_embedding_grad(const void* ids, int id_bytes, int T, int vocab, const void* dy, int dy_dtype, int lddy, int C,
                                    float scale, int64_t padding_idx, float* grad, int ldg, int accumulate, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    if (T < 0 || vocab <= 0 || vocab == 0x7fffffff || C <= 0 || (id_bytes != 4 && id_bytes != 8) || dy_dtype < 0 || dy_dtype > 1 || lddy < C || ldg < C)
        return CCNET_EINVAL;
    if (T > (1 << 30)) return CCNET_EUNSUP;
    const int ds = dy_dtype == 0 ? 4 : 2;
    if (!grad || ((uintptr_t)grad & 3) || (C + 511) / 512 > 65535) return CCNET_EINVAL;
    if (T > 0 && (!ids || !dy || (uintptr_t)ids % id_bytes || (uintptr_t)dy % ds)) return CCNET_EINVAL;
    const Layout l = layout_of(T, vocab, C);
    if (T > 0 && (!workspace || ((uintptr_t)workspace & 15))) return CCNET_EINVAL;
    if (T > 0 && workspace_bytes < l.bytes) return CCNET_EWS;
    if (T == 0 && accumulate) return CCNET_OK;
    hipStream_t st = (hipStream_t)stream;
    char* ws = (char*)workspace;
    GradArgs g{};
    g.T = T; g.vocab = vocab; g.dy = dy; g.lddy = lddy; g.C = C; g.scale = scale; g.grad = grad; g.ldg = ldg; g.accumulate = accumulate != 0;
    if (T > 0) {
        int* keys[2] = {(int*)(ws + l.keys[0]), (int*)(ws + l.keys[1])};
        int* perm[2] = {(int*)(ws + l.perm[0]), (int*)(ws + l.perm[1])};
        g.runs = (i32x2*)(ws + l.runs);
        g.p64 = (float*)(ws + l.p64);
        g.p512 = (float*)(ws + l.p512);
        int cur = 0;
        if (T <= RANK_MOST && vocab < RANK_VOCAB) {
            const int sorting = (T + 63) / 64, clearing = (vocab + 8191) / 8192;
            hipLaunchKernelGGL(rank_sort_kernel, dim3(sorting > clearing ? sorting : clearing), dim3(1024), 0, st, ids, (int)(id_bytes == 8), T, vocab,
                               (long long)padding_idx, keys[0], perm[0], g.runs);
            CCNET_LAUNCH_CHECK();
        } else {
            SortArgs s{};
            s.ids = ids; s.wide = id_bytes == 8; s.T = T; s.vocab = vocab; s.padding = padding_idx; s.hist = (int*)(ws + l.hist); s.runs = g.runs;
            const unsigned blocks = (unsigned)(((long long)T + RS_BLOCK - 1) / RS_BLOCK);
            cur = 1;
            for (int shift = 0; shift < 32 && (vocab >> shift) > 0; shift += 8) {
                s.shift = shift;
                s.keys_out = keys[1 - cur]; s.perm_out = perm[1 - cur];
                hipLaunchKernelGGL(sort_hist_kernel, dim3(blocks), dim3(RS_THREADS), 0, st, s);
                CCNET_LAUNCH_CHECK();
                hipLaunchKernelGGL(sort_scatter_kernel, dim3(blocks), dim3(RS_THREADS), 0, st, s);
                CCNET_LAUNCH_CHECK();
                cur = 1 - cur;
                s.keys_in = keys[cur]; s.perm_in = perm[cur];
            }
        }
        g.keys = keys[cur];
        g.perm = perm[cur];
    }
    const bool vec = C % 8 == 0 && aligned16(dy, lddy, ds) && aligned16(grad, ldg, 4);
    if (dy_dtype == 0) return vec ? launch_grad<float, true>(g, st) : launch_grad<float, false>(g, st);
    return vec ? launch_grad<bf16_t, true>(g, st) : launch_grad<bf16_t, false>(g, st);
}
