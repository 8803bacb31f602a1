// Causal attention over packed prompts (sequences of different lengths end to end in one [rows][channels] matrix), grouped
// heads, head dim 64 or 128, forward and backward, bf16 MFMA with fp32 accumulation and statistics.
//
//   S = scale * q k^T (key <= query, same sequence),  P = softmax(S),  O = P V,  lse = log2 sum_keys 2^(S log2 e)
//   backward, from lse and delta = rowsum(dO o O):  P = 2^(S log2 e - lse),  dS = P o (dO V^T - delta),
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO, the last two summed over the query heads of a key head.
//
// Work is cut into (sequence, 128- or 256-row tile, head); which tile a workgroup takes follows from the offsets in device memory
// (find_tile), so the host needs neither the lengths nor a copy of them, and a captured graph serves other lengths.  The longest
// walks come first.  Rows are addressed relative to their sequence, so the diagonal always falls on aligned 32x32 blocks:
// blocks above it are skipped, blocks on it masked, all others run without a mask.  Rows past a sequence's end are cut off by
// the bounds of the buffer descriptor (read as zero), never by a branch.
//
// Layout of the products (v_mfma_f32_32x32x16_bf16): the forward and dQ kernels keep the QUERY on the lane (S^T = K Q^T, then
// O^T += V^T P^T), the dK / dV kernel the KEY (S = Q K^T, then dV^T += dO^T P): an exponentiated accumulator block, rounded to
// bf16, is then the B operand of the next product as it stands (k order 16 s + 8 (j >> 2) + 4 hh + (j & 3) for element j of
// lane half hh), with the A operand brought in that order by ds_read_b64_tr_b16.  One LDS image serves row reads and transposed
// reads: 16-byte chunk c of row r lies at chunk c ^ swz(r), swz spreading 8 consecutive rows' 64-byte spans as well as 16
// consecutive rows' single chunks evenly over the 64 banks.
#include "common.h"
#include <algorithm>
#include <type_traits>

namespace {

constexpr int PA_TILE = 64;  // rows of a staged tile

struct PackedArgs {
    const __bf16 *Q, *K, *V, *O, *dO;
    __bf16 *out, *dQ, *dK, *dV;
    long long ldq, ldk, ldv, ldo, lddo, lddq, lddk, lddv;
    const int* cu;
    int n_seq, rows, H, Hkv;
    float scale, scale_log2e;
    int zero_tail;  // rows behind the last sequence: 1 = written as zeros, 0 = left as they are
    float* lse;     // [H][rows]
    float* delta;   // [H][rows]
    __bf16* o_low;  // [rows][H d]: what the rounding of O took away
    int skip;       // sequences of at most so many rows have no tiles (packed_bwd_short_kernel takes them)
    int rest, per;  // its workgroups for longer sequences, and how many heads or key heads each takes one after the other
    int parts;      // dK / dV: workgroups that share a key tile's walk, each with H / Hkv / parts query heads
    float* part;    // parts > 1: [parts][2][rows][Hkv d] sums of dK (not scaled yet) and dV
};

template <int D>
__device__ __forceinline__ int swz(int r) {
    if constexpr (D == 64) {
        const int x = (r >> 1) & 7;
        return ((x & 1) << 2) | (x & 2) | (x >> 2);
    } else {
        return ((r & 3) << 2) | ((r >> 2) & 3);
    }
}

__device__ __forceinline__ s16x4 lds_read_tr16(const char* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(p));
}
__device__ __forceinline__ bf16x8 tr_pair(const char* lo_p, const char* hi_p) {
    typedef __attribute__((ext_vector_type(8))) short s16x8;
    const s16x4 lo = lds_read_tr16(lo_p), hi = lds_read_tr16(hi_p);
    return __builtin_bit_cast(bf16x8, s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
}

// 1 KiB of global memory straight to LDS (lane l lands at lds + 16 l).  Written as assembly without a register result: the
// compiler then keeps its own counts for the reads of other stages instead of draining these loads in front of each; the
// kernels wait for them themselves (dma_wait) before the barrier behind which a stage is read.
__device__ __forceinline__ void dma16(const u32x4& rsrc, unsigned lds, unsigned voff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc) : "memory");
}
__device__ __forceinline__ void dma4(const u32x4& rsrc, unsigned lds, unsigned voff) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rsrc) : "memory");
}
// every load of this wave has landed and every LDS read of it has returned, then the workgroup's barrier
__device__ __forceinline__ void stage_fence() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ unsigned lds_addr(const char* p) {
    return (unsigned)(size_t)(__attribute__((address_space(3))) const char*)p;
}
// buffer descriptor over `rows` (<= 96) rows of `width` bytes, `ld` bytes apart: an access behind the last row reads zero
__device__ __forceinline__ u32x4 row_rsrc(const char* base, int rows, long long ld, int width) {
    const unsigned long long p = (unsigned long long)base;
    return u32x4{(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)p), (unsigned)__builtin_amdgcn_readfirstlane((int)((p >> 32) & 0xffffu)),
                 (unsigned)__builtin_amdgcn_readfirstlane(rows > 0 ? (int)((rows - 1) * ld + width) : 0), 0x00020000u};
}

struct Tile { int start, len, tile, ntiles; bool tail; };

// sum and maximum over the wave by row shifts and broadcasts (six vector instructions; a shuffle through LDS takes as long as
// all of them); values are not negative
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, true); }
__device__ __forceinline__ int wave_scan(int v) {  // each lane: the sum up to itself
    v += dpp<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8
    v += dpp<0x112, 0xf>(v);
    v += dpp<0x114, 0xf>(v);
    v += dpp<0x118, 0xf>(v);
    v += dpp<0x142, 0xa>(v);  // row_bcast:15 into rows 1 and 3
    v += dpp<0x143, 0xc>(v);  // row_bcast:31 into rows 2 and 3
    return v;
}
__device__ __forceinline__ int wave_isum(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }
__device__ __forceinline__ int wave_imax(int v) {
    v = max(v, dpp<0x111, 0xf>(v));
    v = max(v, dpp<0x112, 0xf>(v));
    v = max(v, dpp<0x114, 0xf>(v));
    v = max(v, dpp<0x118, 0xf>(v));
    v = max(v, dpp<0x142, 0xa>(v));
    v = max(v, dpp<0x143, 0xc>(v));
    return __builtin_amdgcn_readlane(v, 63);
}

// Tile `idx` of the tiles of `step` rows that the sequences have together, ordered by level: first every sequence's tile with
// the highest level, where a tile's level is its index counted from the end that is walked least.  Tiles of level >= L:
// f(L) = sum_i max(0, ntiles_i - L), falling in L, so a bisection finds the level and a ballot the sequence.  Sequence n_seq
// stands for the rows behind the last one (when they are to be written).  Offsets are clamped to [0, rows] and to rising
// order: wrong ones give wrong results but no access outside.  False: there is no such tile.
// The sums take every workgroup through all offsets, several times.  More than FEW_SEQS sequences are therefore taken in groups of 64:
// the group that begins with sequence i has the places from floor(cu[i] / step) + i on, at least as many as it has tiles, and its
// tiles fill the first of them in order of the sequences (the longest walk of each first, not of all).  The group is found by a search
// of 64 probes a round.  Forward of prompts of up to 77 rows, 8 heads, d 64: 192 of them 16.3 us by the sums, 12.4 by groups, 1024 of
// them 182 / 52; with a sequence of 4096 rows behind 192 of them 59 / 66.  (A place for every sequence instead of every group left
// every second place empty where all have 64 rows, and with it every second CU: 1024 x 64 rows, 16 heads 319 / 189 us.)
constexpr int FEW_SEQS = 127;
template <int step>
__device__ __forceinline__ bool find_place(const PackedArgs& a, int idx, bool from_end, Tile& t) {
    const int lane = threadIdx.x & 63;
    auto at = [&](int i) { return min(max(a.cu[min(i, a.n_seq)], 0), a.rows); };
    int lo = 0, hi = a.n_seq / 64 + 1;  // group lo begins at or in front of idx, group hi behind it
    while (hi - lo > 1) {
        const int n = hi - lo, p = (lo + (int)((long long)n * (lane + 1) / 65)) * 64;
        const int in = __popcll(__ballot(at(p) / step + p <= idx));
        hi = in == 64 ? hi : lo + (int)((long long)n * (in + 1) / 65);
        lo += (int)((long long)n * in / 65);
    }
    const int i = lo * 64 + lane, s = at(i), e = at(i + 1);
    const int len = i > a.n_seq ? 0 : i == a.n_seq ? (a.zero_tail ? a.rows - s : 0) : e - s <= a.skip ? 0 : e - s;
    const int nt = (len + step - 1) / step, upto = wave_scan(nt);
    int k = idx - (__builtin_amdgcn_readlane(s, 0) / step + lo * 64);
    const unsigned long long behind = __ballot(upto > k);
    if (k < 0 || behind == 0) return false;
    const int src = __ffsll(behind) - 1;
    k -= __builtin_amdgcn_readlane(upto - nt, src);
    t.start = __builtin_amdgcn_readlane(s, src);
    t.len = __builtin_amdgcn_readlane(len, src);
    t.ntiles = __builtin_amdgcn_readlane(nt, src);
    t.tail = lo * 64 + src == a.n_seq;
    t.tile = from_end ? k : t.ntiles - 1 - k;
    return true;
}
template <int step>
__device__ __forceinline__ bool find_tile(const PackedArgs& a, int idx, bool from_end, Tile& t) {
    if (a.n_seq > FEW_SEQS) return find_place<step>(a, idx, from_end, t);
    const int lane = threadIdx.x & 63, n = a.n_seq + 1;
    auto span = [&](int i, int& s) {
        if (i >= n) { s = 0; return 0; }
        s = min(max(a.cu[i], 0), a.rows);
        const int e = i < a.n_seq ? min(max(a.cu[i + 1], s), a.rows) : (a.zero_tail ? a.rows : s);
        return i < a.n_seq && e - s <= a.skip ? 0 : e - s;
    };
    int s0;
    const int len0 = span(lane, s0), nt0 = (len0 + step - 1) / step;  // the first 64 sequences stay in registers
    auto total = [&](int L) {
        int v = max(0, nt0 - L);
        for (int i = lane + 64; i < n; i += 64) {
            int s;
            v += max(0, (span(i, s) + step - 1) / step - L);
        }
        return wave_isum(v);
    };
    if (total(0) <= idx) return false;
    int m = nt0;
    for (int i = lane + 64; i < n; i += 64) {
        int s;
        m = max(m, (span(i, s) + step - 1) / step);
    }
    int lo = 0, hi = wave_imax(m);  // f(lo) > idx >= f(hi) = 0
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (total(mid) > idx) lo = mid;
        else hi = mid;
    }
    int rank = idx - total(lo + 1);
    for (int i0 = 0; i0 < n; i0 += 64) {
        int s = s0, len = len0;
        if (i0 > 0) len = span(i0 + lane, s);
        const int nt = (len + step - 1) / step;
        const unsigned long long has = __ballot(nt > lo);
        const int c = __popcll(has);
        if (rank < c) {
            const int mine = __popcll(has & ((1ull << lane) - 1));
            const unsigned long long pick = __ballot(nt > lo && mine == rank);
            const int src = __ffsll((unsigned long long)pick) - 1;
            t.start = __builtin_amdgcn_readlane(s, src);
            t.len = __builtin_amdgcn_readlane(len, src);
            t.ntiles = __builtin_amdgcn_readlane(nt, src);
            t.tile = from_end ? t.ntiles - 1 - lo : lo;
            t.tail = i0 + src == a.n_seq;
            return true;
        }
        rank -= c;
    }
    return false;
}

// Consecutive workgroups go to the 8 XCDs in turn: with at least 8 key heads, workgroup slot s of a tile takes key head s mod 8
// (+ 8 ...), so that an XCD's L2 sees the keys and values of its own heads only, all their query heads in turn.
__device__ __forceinline__ int head_of_slot(int s, int H, int Hkv) {
    if (Hkv & 7) return s;
    const int G = H / Hkv, i = s >> 3;
    return ((s & 7) + 8 * (i / G)) * G + i % G;
}

// A value that is not finite must reach only the queries that see its key, but 0 * inf in the product is no zero.  On the
// diagonal block such values are taken out of the operand (finite_part) and, after the walk, put in by hand (add_nonfinite): a
// query gets an infinity or a NaN in a channel from the first key on that holds one there.
__device__ __forceinline__ u32x4 finite_part(const u32x4& f, bool& bad) {
    u32x4 r;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        unsigned v = f[w];
        if ((f[w] & 0x7f80u) == 0x7f80u) v &= 0xffff0000u;
        if ((f[w] & 0x7f800000u) == 0x7f800000u) v &= 0xffffu;
        bad |= v != f[w];
        r[w] = v;
    }
    return r;
}
// o: block of 32 channels x 32 queries (query l31 on the lane); v: the value of channel l31 at the block's first key
__device__ __forceinline__ void add_nonfinite(f32x16& o, const __bf16* v, long long ldv, int keys, int l31, int hh) {
    int pos = 32, neg = 32, nan = 32;
    for (int k = keys - 1; k >= 0; --k) {
        const unsigned b = *(const unsigned short*)(v + k * ldv);
        if ((b & 0x7f80u) != 0x7f80u) continue;
        if (b & 0x7fu) nan = k;
        else if (b >> 15) neg = k;
        else pos = k;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const int c = (e & 3) + 8 * (e >> 2) + 4 * hh;
        if (__shfl(pos, c) <= l31) o[e] += INFINITY;
        if (__shfl(neg, c) <= l31) o[e] -= INFINITY;
        if (__shfl(nan, c) <= l31) o[e] += NAN;
    }
}

// lane addresses of the two transposed 8-byte reads (rows 4 hh + tq and + 8) that fill the A operand of 32-channel block d
template <int D>
__device__ __forceinline__ void tr_lane(int lane, int d, int& lo, int& hi) {
    const int hh = lane >> 5, g16 = (lane >> 4) & 1, tq = (lane & 15) >> 2, tp = lane & 3;
    const int chunk = d * 4 + g16 * 2 + (tp >> 1), r = 4 * hh + tq;
    lo = r * D * 2 + ((chunk ^ swz<D>(r)) << 4) + (tp & 1) * 8;
    hi = (r + 8) * D * 2 + ((chunk ^ swz<D>(r + 8)) << 4) + (tp & 1) * 8;
}

// the DMA pieces of a tile that a wave brings: piece p holds 1024 / (2 D) rows, lane l of it chunk position l mod (D / 8)
template <int D, int W, int ROWS = PA_TILE>
struct TileDma {
    static constexpr int ROWB = 2 * D, CH = D / 8, BYTES = ROWS * ROWB, PIECES = BYTES / 1024 / W;
    static_assert(BYTES % (1024 * W) == 0, "whole pieces a wave");
    unsigned voff[PIECES];
    int wave;
    __device__ __forceinline__ void init(int wave_, int lane, long long ldb) {
        wave = wave_;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            const int r = (wave * PIECES + i) * (1024 / ROWB) + lane / CH, c = (lane % CH) ^ swz<D>(r);
            voff[i] = (unsigned)r * (unsigned)ldb + c * 16;
        }
    }
    __device__ __forceinline__ void issue(const u32x4& rsrc, unsigned lds) const {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) dma16(rsrc, lds + (wave * PIECES + i) * 1024, voff[i]);
    }
};

// a lane's row of `D` values as B-operand fragments (lane: row, half hh: channels 16 ks + 8 hh .. + 7); zeros where !ok
template <int D>
__device__ __forceinline__ void load_frags(bf16x8* f, const __bf16* row, int hh, bool ok) {
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
        u32x4 v = {0u, 0u, 0u, 0u};
        if (ok) v = *(const u32x4*)(row + ks * 16 + hh * 8);
        f[ks] = __builtin_bit_cast(bf16x8, v);
    }
}

// Values that the compiler has loaded from memory are in their registers from here on: without this it would wait for them at
// their first use, inside the walk, on every round, and drain the tile in flight with them.
template <int N>
__device__ __forceinline__ void settle(bf16x8 (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
}

// a lane's row of an accumulator (register e of block d: channel 32 d + (e & 3) + 8 (e >> 2) + 4 hh) as 16-byte stores: the
// swap of packed quads between the lane halves leaves 8 consecutive channels in each
__device__ __forceinline__ u32x4 swap_quads(const unsigned (&p)[4]) {
    u32x4 v;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
        const auto sw = __builtin_amdgcn_permlane32_swap(p[w], p[2 + w], false, false);
        v[w] = sw[0];
        v[2 + w] = sw[1];
    }
    return v;
}
template <int D>
__device__ __forceinline__ void store_row(__bf16* row, __bf16* low_row, const f32x16* o, float mul, int hh, bool ok) {
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int qp = 0; qp < 2; ++qp) {
            unsigned hi[4], lo[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float a = o[d][8 * qp + 2 * w] * mul, b = o[d][8 * qp + 2 * w + 1] * mul;
                hi[w] = pack_bf16x2(a, b);
                lo[w] = pack_bf16x2(a - __uint_as_float(hi[w] << 16), b - __uint_as_float(hi[w] & 0xffff0000u));
            }
            const u32x4 v = swap_quads(hi);
            if (ok) *(u32x4*)(row + d * 32 + 16 * qp + 8 * hh) = v;
            if (low_row) {
                const u32x4 r = swap_quads(lo);
                if (ok) *(u32x4*)(low_row + d * 32 + 16 * qp + 8 * hh) = r;
            }
        }
}

// what the rounding of f to the bf16 of `hi` took away, rounded itself.  (Where f is a product, the compiler would fuse it with the
// difference in some of the kernels and not in others, whose results then differ in a last bit here and there.)
__device__ __forceinline__ u32x4 rounded_off(const float (&f)[8], const u32x4& hi) {
#pragma clang fp contract(off)
    float r[8];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        r[2 * w] = f[2 * w] - __uint_as_float(hi[w] << 16);
        r[2 * w + 1] = f[2 * w + 1] - __uint_as_float(hi[w] & 0xffff0000u);
    }
    return pack8(r);
}

__device__ __forceinline__ float half_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// ------------------------------------------------------------------ forward
// A wave owns QB blocks of 32 queries and walks the keys in blocks of 32, staged as tiles of 64.  Step j of the walk takes the
// scores of key block j, which the step before has left, through the softmax and into O, and computes the scores of block
// j + 1 beside it: the two products of a step and its exponentials are independent, so that the matrix pipe and the vector
// pipe, which need about 512 cycles a step each at d = 128, run at once.  Half way through a tile's two steps lies the fence at
// which the next tile has landed (its keys are needed by the second step) and the tile after it is sent for: K in a ring of
// two, V, which is needed a step longer, in a ring of three.
// Bound by both pipes' issue at d = 128 (4 sequences of 2811 to 8192 rows, 32 / 8 heads: 862 to 883 us = 990 to 1015 TFLOP/s, a square
// product of 16384 reaches 1364; counters at 5 sequences of 1528 to 4096 rows: the matrix pipe busy 0.44 of the time, the vector pipe
// 0.49), by vector issue at d = 64, where every product has half the work an exponential (those 5, 16 / 4 heads: 114 us = 750 TFLOP/s with
// the statistics for the backward; vector pipe 0.67, matrix pipe 0.36, a CU without work 0.16), by latency for prompts (77 rows, 16 heads:
// 5.9 us; 32 prompts 6.6 us; 4096 of up to 77 rows: 484 us, 578 with the statistics; matrix pipe 0.04, half of the waves' time waits).
template <int D, int QB, int W>
__global__ __launch_bounds__(64 * W, 2) void packed_fwd_kernel(const PackedArgs a) {
    constexpr int BM = 32 * W * QB, NK = D / 16, ND = D / 32, ROWB = 2 * D, TILEB = PA_TILE * ROWB, BLOCKB = 32 * ROWB;
    __shared__ __attribute__((aligned(1024))) char smem[5 * TILEB];  // K 0, K 1, V 0, V 1, V 2
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l31 = lane & 31, hh = lane >> 5;
    Tile tl;
    if (!find_tile<BM>(a, blockIdx.x / a.H, false, tl)) return;
    const int h = head_of_slot(blockIdx.x % a.H, a.H, a.Hkv), kvh = h / (a.H / a.Hkv);
    const int q0 = tl.tile * BM + wave * 32 * QB;  // in the sequence

    f32x16 o[QB][ND];
    float m_run[QB], l_run[QB];
#pragma unroll
    for (int X = 0; X < QB; ++X) {
        m_run[X] = -INFINITY;
        l_run[X] = 0.f;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[X][d][e] = 0.f;
    }
    if (!tl.tail) {
        bf16x8 qf[QB][NK];
#pragma unroll
        for (int X = 0; X < QB; ++X) {
            const int q = q0 + 32 * X + l31;
            load_frags<D>(qf[X], a.Q + (long long)(tl.start + min(q, tl.len - 1)) * a.ldq + h * D, hh, q < tl.len);
        }
        const long long ldkb = a.ldk * 2, ldvb = a.ldv * 2;
        const char* kbase = (const char*)(a.K + (long long)tl.start * a.ldk + kvh * D);
        const char* vbase = (const char*)(a.V + (long long)tl.start * a.ldv + kvh * D);
        TileDma<D, W> kd, vd;
        kd.init(wave, lane, ldkb);
        vd.init(wave, lane, ldvb);
        const unsigned lds0 = lds_addr(smem);
        auto issue = [&](int t, int vslot) {
            const int left = min(tl.len - t * PA_TILE, PA_TILE);
            kd.issue(row_rsrc(kbase + (long long)t * PA_TILE * ldkb, left, ldkb, ROWB), lds0 + (t & 1) * TILEB);
            vd.issue(row_rsrc(vbase + (long long)t * PA_TILE * ldvb, left, ldvb, ROWB), lds0 + (2 + vslot) * TILEB);
        };
        int kread[NK], vlo[ND], vhi[ND];
#pragma unroll
        for (int ks = 0; ks < NK; ++ks) kread[ks] = l31 * ROWB + (((2 * ks + hh) ^ swz<D>(l31)) << 4);
#pragma unroll
        for (int d = 0; d < ND; ++d) tr_lane<D>(lane, d, vlo[d], vhi[d]);

        f32x16 s[QB];
        auto scores = [&](f32x16 (&r)[QB], const char* kb, int X0) {  // of query blocks X0 .. with the key block at kb
#pragma unroll
            for (int X = X0; X < QB; ++X)
#pragma unroll
                for (int e = 0; e < 16; ++e) r[X][e] = 0.f;
#pragma unroll
            for (int ks = 0; ks < NK; ++ks) {
                const bf16x8 kf = *(const bf16x8*)(kb + kread[ks]);
#pragma unroll
                for (int X = X0; X < QB; ++X) r[X] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[X][ks], r[X], 0, 0, 0);
            }
        };
        bool bad = false;  // a value on this wave's diagonal that is not finite
        // One step: vb = V of this key block, kn = K of the next.  X0: first query block that sees this key block; diag: the query
        // block on the diagonal (-1: none); XN: first query block that sees the next one (QB: there is no next).
        auto step = [&](const char* vb, const char* kn, auto x0_c, auto diag_c, auto xn_c) {
            constexpr int X0 = decltype(x0_c)::value, DIAG = decltype(diag_c)::value, XN = decltype(xn_c)::value;
            if constexpr (DIAG >= 0) {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if ((e & 3) + 8 * (e >> 2) + 4 * hh > l31) s[DIAG][e] = -INFINITY;
            }
            // running maximum in the scaled log2 domain; kept while no row of the wave outgrows it by more than 2^6, so that the
            // rescaling of O and l is rare (P <= 64 stays exact in fp32, and its rounding to bf16 is relative)
            float mx[QB];
            bool grew = false;
#pragma unroll
            for (int X = X0; X < QB; ++X) {
                float m = -INFINITY;
#pragma unroll
                for (int e = 0; e < 16; ++e) m = fmaxf(m, s[X][e]);
                mx[X] = half_max(m) * a.scale_log2e;
                grew |= !(mx[X] - m_run[X] <= 6.0f);
            }
            if (__any(grew)) {
#pragma unroll
                for (int X = X0; X < QB; ++X) {
                    const float m_new = fmaxf(m_run[X], mx[X]);
                    // a row that has seen only -inf scores keeps -inf as its maximum; its l stays 0 and its result 0 / 0
                    const float alpha = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_run[X] - m_new);
                    m_run[X] = m_new;
                    l_run[X] *= alpha;
#pragma unroll
                    for (int d = 0; d < ND; ++d)
#pragma unroll
                        for (int e = 0; e < 16; ++e) o[X][d][e] *= alpha;
                }
            }
            f32x16 sn[QB];
            if constexpr (XN < QB) scores(sn, kn, XN);
            u32x4 pf[QB][2];
#pragma unroll
            for (int X = X0; X < QB; ++X) {
                const float m = m_run[X] == -INFINITY ? 0.f : m_run[X];
#pragma unroll
                for (int sI = 0; sI < 2; ++sI) {
                    float p[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) p[j] = __builtin_amdgcn_exp2f(fmaf(s[X][8 * sI + j], a.scale_log2e, -m));
                    l_run[X] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
                    pf[X][sI] = pack8(p);
                }
            }
            u32x4 vf[ND][2];
#pragma unroll
            for (int sI = 0; sI < 2; ++sI)
#pragma unroll
                for (int d = 0; d < ND; ++d)
                    vf[d][sI] = __builtin_bit_cast(u32x4, tr_pair(vb + sI * 16 * ROWB + vlo[d], vb + sI * 16 * ROWB + vhi[d]));
            auto pv = [&](int X) {
#pragma unroll
                for (int sI = 0; sI < 2; ++sI)
#pragma unroll
                    for (int d = 0; d < ND; ++d)
                        o[X][d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, vf[d][sI]), __builtin_bit_cast(bf16x8, pf[X][sI]),
                                                                         o[X][d], 0, 0, 0);
            };
#pragma unroll
            for (int X = X0; X < QB; ++X)
                if (X != DIAG) pv(X);
            if constexpr (DIAG >= 0) {
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int sI = 0; sI < 2; ++sI) vf[d][sI] = finite_part(vf[d][sI], bad);
                pv(DIAG);
            }
            if constexpr (XN < QB) {
#pragma unroll
                for (int X = XN; X < QB; ++X) s[X] = sn[X];
            }
        };
        using zero = std::integral_constant<int, 0>;
        using one = std::integral_constant<int, 1>;
        using none = std::integral_constant<int, -1>;
        using end = std::integral_constant<int, QB>;
        // keys that the workgroup sees: up to its last query; the wave's diagonal lies in key block jd
        const int ntiles = (min((tl.tile + 1) * BM, tl.len) + PA_TILE - 1) / PA_TILE;
        const int jd = q0 / 32, walk = q0 < tl.len ? jd / 2 : 0;  // tiles that the wave takes whole
        issue(0, 0);
#pragma unroll
        for (int X = 0; X < QB; ++X) settle(qf[X]);
        if (ntiles > 1) {
            issue(1, 1);
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * TileDma<D, W>::PIECES) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        }
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        int v = 0, t = 0;  // ring slot of the tile's values, tile
        auto fence = [&]() {  // tile t + 1 has landed, and what tile t + 2 overwrites is no longer read
            stage_fence();
            if (t + 2 < ntiles) issue(t + 2, v == 0 ? 2 : v - 1);
        };
        if (q0 < tl.len) scores(s, smem, 0);
        for (; t < walk; ++t) {
            const char* vb = smem + (2 + v) * TILEB;
            step(vb, smem + (t & 1) * TILEB + BLOCKB, zero{}, none{}, zero{});
            fence();
            step(vb + BLOCKB, smem + ((t + 1) & 1) * TILEB, zero{}, none{}, zero{});
            v = v == 2 ? 0 : v + 1;
        }
        if (q0 < tl.len) {  // the tile that holds the diagonal, in its first block or (QB 1, every other wave) its second
            const char* vb = smem + (2 + v) * TILEB;
            const char* kn = smem + (t & 1) * TILEB + BLOCKB;
            if constexpr (QB == 2) {
                step(vb, kn, zero{}, zero{}, one{});
                fence();
                step(vb + BLOCKB, kn, one{}, one{}, end{});
            } else if (jd & 1) {
                step(vb, kn, zero{}, none{}, zero{});
                fence();
                step(vb + BLOCKB, kn, zero{}, zero{}, end{});
            } else {
                step(vb, kn, zero{}, zero{}, end{});
                fence();
            }
            v = v == 2 ? 0 : v + 1;
            ++t;
        }
        for (; t < ntiles; ++t, v = v == 2 ? 0 : v + 1) fence();
        if (__any(bad)) {
#pragma unroll
            for (int X = 0; X < QB; ++X) {
                const int k0 = q0 + 32 * X;
#pragma unroll
                for (int d = 0; d < ND; ++d)
                    add_nonfinite(o[X][d], a.V + (long long)(tl.start + k0) * a.ldv + kvh * D + d * 32 + l31, a.ldv, min(tl.len - k0, 32), l31, hh);
            }
        }
    }
#pragma unroll
    for (int X = 0; X < QB; ++X) {
        const int q = q0 + 32 * X + l31;
        const bool ok = q < tl.len;
        const float l = half_sum(l_run[X]);
        if (a.lse && hh == 0 && ok) a.lse[(long long)h * a.rows + tl.start + q] = tl.tail ? -INFINITY : m_run[X] + __builtin_amdgcn_logf(l);
        const long long row = tl.start + (ok ? q : 0);
        store_row<D>(a.out + row * a.ldo + h * D, a.o_low ? a.o_low + (row * a.H + h) * D : nullptr, o[X], tl.tail ? 0.f : 1.0f / l, hh, ok);
    }
}

// Where dP begins: at -delta, or at zero with -delta added to the product (the first spills in dQ at d 128); the same to the bit in all
// of the backward's kernels, so that which of them takes a sequence does not show.  (Into how many parts a key head's walk is cut does,
// in the last bits of dK and dV: parts_of.)
template <int D>
constexpr bool FROM_DELTA = D == 64;
__device__ __forceinline__ void add_delta(f32x16& dp, const float* delta, int hh) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const f32x4 d4 = *(const f32x4*)(delta + 8 * g + 4 * hh);
#pragma unroll
        for (int j = 0; j < 4; ++j) dp[4 * g + j] += d4[j];
    }
}

// ------------------------------------------------------------------ backward: dQ (and delta)
// The forward's walk with 32 queries a wave: S^T = K Q^T and dP^T = V dO^T from row reads, a block ahead of dQ^T += K^T dS^T
// from transposed reads, so here K is needed a step longer (ring of three).  delta is taken from the wave's own dO and O rows
// and left for the dK / dV kernel.  Bound by matrix and vector issue side by side: 13.6k rows, 16 / 4 heads, d 64: 149 to 154 us =
// 830 to 860 TFLOP/s of its three products (a twelfth more are for dS's low parts); matrix pipe busy 0.45, vector pipe 0.52; at d 128
// 279 to 286 us, 0.48 and 0.39.
template <int D, int W>
__device__ __forceinline__ void dq_walk(const PackedArgs& a, const Tile& tl, int h, char* smem) {
    constexpr int BM = 32 * W, NK = D / 16, ND = D / 32, ROWB = 2 * D, TILEB = PA_TILE * ROWB, BLOCKB = 32 * ROWB;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l31 = lane & 31, hh = lane >> 5;
    const int kvh = h / (a.H / a.Hkv);
    const int q0 = tl.tile * BM + wave * 32, q = q0 + l31;
    const bool qok = q < tl.len;
    const long long row = tl.start + (qok ? q : 0);
    f32x16 dq[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) dq[d][e] = 0.f;
    if (!tl.tail) {
        bf16x8 qf[NK], dof[NK];
        load_frags<D>(qf, a.Q + row * a.ldq + h * D, hh, qok);
        load_frags<D>(dof, a.dO + row * a.lddo + h * D, hh, qok);
        const long long ldkb = a.ldk * 2, ldvb = a.ldv * 2;
        const char* kbase = (const char*)(a.K + (long long)tl.start * a.ldk + kvh * D);
        const char* vbase = (const char*)(a.V + (long long)tl.start * a.ldv + kvh * D);
        TileDma<D, W> kd, vd;
        kd.init(wave, lane, ldkb);
        vd.init(wave, lane, ldvb);
        const unsigned lds0 = lds_addr(smem);
        auto issue = [&](int t, int kslot) {
            const int left = min(tl.len - t * PA_TILE, PA_TILE);
            kd.issue(row_rsrc(kbase + (long long)t * PA_TILE * ldkb, left, ldkb, ROWB), lds0 + (2 + kslot) * TILEB);
            vd.issue(row_rsrc(vbase + (long long)t * PA_TILE * ldvb, left, ldvb, ROWB), lds0 + (t & 1) * TILEB);
        };
        issue(0, 0);
        float dlt = 0.f;
#pragma unroll
        for (int ks = 0; ks < NK; ++ks) {
            u32x4 ov = {0u, 0u, 0u, 0u}, lv = {0u, 0u, 0u, 0u};
            if (qok) ov = *(const u32x4*)(a.O + row * a.ldo + h * D + ks * 16 + hh * 8);
            if (qok && a.o_low) lv = *(const u32x4*)(a.o_low + (row * a.H + h) * D + ks * 16 + hh * 8);
            float x[8], l[8], y[8];
            unpack8(ov, x);
            unpack8(lv, l);
            unpack8(__builtin_bit_cast(u32x4, dof[ks]), y);
#pragma unroll
            for (int j = 0; j < 8; ++j) dlt = fmaf(x[j] + l[j], y[j], dlt);
        }
        dlt = -half_sum(dlt);  // (negative: where dP starts from)
        if (hh == 0 && qok) a.delta[(long long)h * a.rows + row] = dlt;
        float lse = qok ? a.lse[(long long)h * a.rows + row] : 0.f;
        int rread[NK], klo[ND], khi[ND];
#pragma unroll
        for (int ks = 0; ks < NK; ++ks) rread[ks] = l31 * ROWB + (((2 * ks + hh) ^ swz<D>(l31)) << 4);
#pragma unroll
        for (int d = 0; d < ND; ++d) tr_lane<D>(lane, d, klo[d], khi[d]);
        const int last = q == 0 ? -1 : l31;  // the last key of the diagonal block whose dS counts: query 0 sees one key, P = 1, dS = 0
        f32x16 s, dp;
        auto scores = [&](f32x16& sr, f32x16& dr, const char* kb, const char* vb) {
#pragma unroll
            for (int e = 0; e < 16; ++e) { sr[e] = 0.f; dr[e] = FROM_DELTA<D> ? dlt : 0.f; }
#pragma unroll
            for (int ks = 0; ks < NK; ++ks) {
                sr = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(kb + rread[ks]), qf[ks], sr, 0, 0, 0);
                dr = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(vb + rread[ks]), dof[ks], dr, 0, 0, 0);
            }
        };
        // kb: K of this key block; kn, vn: K and V of the next.  MORE (every other block): what the rounding of dS to bf16 takes away from
        // the block's first 16 keys goes into a second product.  Without it dQ is 1.5 times as far from the exact one as its own rounding to
        // bf16 brings it; with it for these keys 1.4 times, or 1.1 for prompts (backward of 13.6k rows, 16 / 4 heads: 330 -> 344 us), for
        // half of them 1.3 (353), for all 1.1 (369).
        auto step = [&](const char* kb, const char* kn, const char* vn, auto diag_c, auto next_c, auto more_c) {
            constexpr bool DIAG = decltype(diag_c)::value, NEXT = decltype(next_c)::value, MORE = decltype(more_c)::value;
            f32x16 sn, dpn;
            if constexpr (NEXT) scores(sn, dpn, kn, vn);
            bf16x8 dsf[2], low;
            auto terms = [&](int sI) {
                float ds[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int e = 8 * sI + j;
                    ds[j] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale_log2e, -lse)) * (FROM_DELTA<D> ? dp[e] : dp[e] + dlt);
                    if (DIAG && (e & 3) + 8 * (e >> 2) + 4 * hh > last) ds[j] = 0.f;
                }
                const u32x4 hi = pack8(ds);
                dsf[sI] = __builtin_bit_cast(bf16x8, hi);
                if (MORE && sI == 0) low = __builtin_bit_cast(bf16x8, rounded_off(ds, hi));
            };
            auto products = [&](int sI) {
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const bf16x8 kt = tr_pair(kb + sI * 16 * ROWB + klo[d], kb + sI * 16 * ROWB + khi[d]);
                    dq[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kt, dsf[sI], dq[d], 0, 0, 0);
                    if (MORE && sI == 0) dq[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kt, low, dq[d], 0, 0, 0);
                }
            };
            terms(0);
            if constexpr (D == 128) {  // (the other order spills)
                products(0);
                terms(1);
            } else {
                terms(1);
                products(0);
            }
            products(1);
            if constexpr (NEXT) { s = sn; dp = dpn; }
        };
        const int ntiles = (min((tl.tile + 1) * BM, tl.len) + PA_TILE - 1) / PA_TILE;
        const int jd = q0 / 32, walk = q0 < tl.len ? jd / 2 : 0;
        settle(qf);
        settle(dof);
        asm volatile("" : "+v"(lse), "+v"(dlt));
        if (ntiles > 1) {
            issue(1, 1);
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(2 * TileDma<D, W>::PIECES) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        }
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        int kslot = 0, t = 0;
        auto next_slot = [&]() { return kslot == 2 ? 0 : kslot + 1; };
        auto fence = [&]() {  // tile t + 1 has landed, and what tile t + 2 overwrites is no longer read
            stage_fence();
            if (t + 2 < ntiles) issue(t + 2, kslot == 0 ? 2 : kslot - 1);
        };
        if (q0 < tl.len) scores(s, dp, smem + 2 * TILEB, smem);
        for (; t < walk; ++t) {
            const char* kb = smem + (2 + kslot) * TILEB;
            step(kb, kb + BLOCKB, smem + (t & 1) * TILEB + BLOCKB, std::false_type{}, std::true_type{}, std::true_type{});
            fence();
            step(kb + BLOCKB, smem + (2 + next_slot()) * TILEB, smem + ((t + 1) & 1) * TILEB, std::false_type{}, std::true_type{}, std::false_type{});
            kslot = next_slot();
        }
        if (q0 < tl.len) {
            const char* kb = smem + (2 + kslot) * TILEB;
            if (jd & 1) {
                step(kb, kb + BLOCKB, smem + (t & 1) * TILEB + BLOCKB, std::false_type{}, std::true_type{}, std::true_type{});
                fence();
                step(kb + BLOCKB, nullptr, nullptr, std::true_type{}, std::false_type{}, std::false_type{});
            } else {
                step(kb, nullptr, nullptr, std::true_type{}, std::false_type{}, std::true_type{});
                fence();
            }
            kslot = next_slot();
            ++t;
        }
        for (; t < ntiles; ++t, kslot = next_slot()) fence();
    }
    store_row<D>(a.dQ + row * a.lddq + h * D, nullptr, dq, a.scale, hh, qok);
}

template <int D, int W>
__global__ __launch_bounds__(64 * W, 2) void packed_bwd_dq_kernel(const PackedArgs a) {
    __shared__ __attribute__((aligned(1024))) char smem[5 * PA_TILE * 2 * D];  // V 0, V 1, K 0, K 1, K 2
    Tile tl;
    if (find_tile<32 * W>(a, blockIdx.x / a.H, false, tl)) dq_walk<D, W>(a, tl, head_of_slot(blockIdx.x % a.H, a.H, a.Hkv), smem);
}

// ------------------------------------------------------------------ backward: dK, dV
// A wave owns 32 keys of a key head; the workgroup walks the query tiles from its own diagonal on, for the query heads of the
// group (or of its part of it) in turn, so the group's sum is taken in the accumulators, in a fixed order.  As above the scores
// of the next query block are computed beside the exponentials of this one; Q and dO are both needed a step longer (rings of
// three).  Query blocks in front of a wave's own keys (in the first two tiles of a head) are masked whole.
// Bound like dQ, two workgroups a CU both: the same 13.6k rows 195 to 200 us = 850 to 875 TFLOP/s of its four products; matrix pipe busy
// 0.47, vector pipe 0.41, LDS 0.33.  At d 128 (430 registers, 99,840 bytes) one workgroup a CU, so one wave a SIMD and nothing beside it
// while it waits: 410 to 437 us, matrix pipe 0.39, vector pipe 0.29.
template <int D>
constexpr int dkv_stage() { return 2 * PA_TILE * 2 * D + 512; }  // Q, dO, lse and delta of 64 queries
template <int D, int W>
__device__ __forceinline__ void dkv_walk(const PackedArgs& a, const Tile& tl, int kvh, int part, char* smem) {
    constexpr int BM = 32 * W, NK = D / 16, ND = D / 32, ROWB = 2 * D, TILEB = PA_TILE * ROWB, BLOCKB = 32 * ROWB, STAGEB = dkv_stage<D>();
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l31 = lane & 31, hh = lane >> 5;
    const int G = a.H / a.Hkv / a.parts, h0 = (kvh * a.parts + part) * G;
    const int k0 = tl.tile * BM + wave * 32, key = k0 + l31;
    const bool kok = key < tl.len;
    const long long row = tl.start + (kok ? key : 0);
    f32x16 dk[ND], dv[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) { dk[d][e] = 0.f; dv[d][e] = 0.f; }
    if (!tl.tail) {
        bf16x8 kf[NK], vf[NK];
        load_frags<D>(kf, a.K + row * a.ldk + kvh * D, hh, kok);
        load_frags<D>(vf, a.V + row * a.ldv + kvh * D, hh, kok);
        const long long ldqb = a.ldq * 2, lddob = a.lddo * 2;
        TileDma<D, W> qd, dd;
        qd.init(wave, lane, ldqb);
        dd.init(wave, lane, lddob);
        const unsigned lds0 = lds_addr(smem);
        const int t0 = tl.tile * BM / PA_TILE, per_head = (tl.len + PA_TILE - 1) / PA_TILE - t0, steps = per_head * G;
        int ig = 0, it = 0, islot = 0, issued = 0;  // next tile to send for: head of the part, tile behind t0, ring slot
        auto issue = [&]() {
            if (issued == steps) return;
            const int h = h0 + ig, t = t0 + it, left = min(tl.len - t * PA_TILE, PA_TILE);
            const long long r0 = (long long)tl.start + t * PA_TILE;
            const unsigned st = lds0 + islot * STAGEB;
            qd.issue(row_rsrc((const char*)(a.Q + r0 * a.ldq + h * D), left, ldqb, ROWB), st);
            dd.issue(row_rsrc((const char*)(a.dO + r0 * a.lddo + h * D), left, lddob, ROWB), st + TILEB);
            if (wave < 2) {  // queries behind the end read as lse = delta = 0, q = dO = 0: P = 1 meets only zeros
                const float* p = (wave == 0 ? a.lse : a.delta) + (long long)h * a.rows + r0;
                dma4(row_rsrc((const char*)p, left, 4, 4), st + 2 * TILEB + wave * 256, lane * 4);
            }
            ++issued;
            islot = islot == 2 ? 0 : islot + 1;
            if (++it == per_head) { it = 0; ++ig; }
        };
        int rread[NK], tlo[ND], thi[ND];
#pragma unroll
        for (int ks = 0; ks < NK; ++ks) rread[ks] = l31 * ROWB + (((2 * ks + hh) ^ swz<D>(l31)) << 4);
#pragma unroll
        for (int d = 0; d < ND; ++d) tr_lane<D>(lane, d, tlo[d], thi[d]);
        f32x16 s, dp;
        // fragments of the next block's rows (fq, fd) and of this block's transposed reads (tq, td) are read a phase ahead of the
        // products that take them
        bf16x8 fq[NK], fd[NK], tq[2][ND], td[2][ND];
        auto rows = [&](const char* qb) {
#pragma unroll
            for (int ks = 0; ks < NK; ++ks) {
                fq[ks] = *(const bf16x8*)(qb + rread[ks]);
                fd[ks] = *(const bf16x8*)(qb + TILEB + rread[ks]);
            }
        };
        auto scores = [&](f32x16& sr, f32x16& dr, const float* stat) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 d4 = *(const f32x4*)(stat + 64 + 8 * g + 4 * hh);
#pragma unroll
                for (int j = 0; j < 4; ++j) { sr[4 * g + j] = 0.f; dr[4 * g + j] = FROM_DELTA<D> ? d4[j] : 0.f; }
            }
#pragma unroll
            for (int ks = 0; ks < NK; ++ks) {
                sr = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fq[ks], kf[ks], sr, 0, 0, 0);
                dr = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fd[ks], vf[ks], dr, 0, 0, 0);
            }
        };
        // MORE (every other block): as in dQ, for the block's first 16 queries (dK 1.45 to 1.7 -> 1.1 to 1.4 times its own rounding;
        // backward of 13.6k rows 350 -> 360 us).
        // qb: Q of this query block (dO a tile behind it), stat: its lse, rel: its index counted from the wave's diagonal, statn: of
        // the next block, qnn: Q of the block after that
        auto step = [&](const char* qb, const float* stat, int rel, const float* statn, const char* qnn, auto fence_c) {
            if constexpr (!FROM_DELTA<D>) add_delta(dp, stat + 64, hh);
            if (rel <= 0) {
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (rel * 32 + (e & 3) + 8 * (e >> 2) + 4 * hh < l31) s[e] = -INFINITY;  // P = 0, dS = 0
                if (rel == 0 && k0 + hh == 0) dp[0] = 0.f;                                // (query 0 sees one key: P = 1, dS = 0)
            }
            f32x16 sn, dpn;
            scores(sn, dpn, statn);
            constexpr bool MORE = decltype(fence_c)::value;
            bf16x8 pfr[2], dsf[2], low;
#pragma unroll
            for (int sI = 0; sI < 2; ++sI) {
                float p[8], ds[8];
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const int qo = 16 * sI + 8 * g + 4 * hh;  // registers 8 sI + 4 g .. + 3: four consecutive queries
                    const f32x4 l4 = *(const f32x4*)(stat + qo);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int e = 8 * sI + 4 * g + j;
                        p[4 * g + j] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale_log2e, -l4[j]));
                        ds[4 * g + j] = p[4 * g + j] * dp[e];
                    }
                }
                pfr[sI] = __builtin_bit_cast(bf16x8, pack8(p));
                const u32x4 hi = pack8(ds);
                dsf[sI] = __builtin_bit_cast(bf16x8, hi);
                if (MORE && sI == 0) low = __builtin_bit_cast(bf16x8, rounded_off(ds, hi));
            }
#pragma unroll
            for (int sI = 0; sI < 2; ++sI)
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const char* x = qb + sI * 16 * ROWB;
                    td[sI][d] = tr_pair(x + TILEB + tlo[d], x + TILEB + thi[d]);
                    tq[sI][d] = tr_pair(x + tlo[d], x + thi[d]);
                }
            if constexpr (decltype(fence_c)::value) {
                stage_fence();  // the next tile has landed; the tile after it may overwrite the one before this
                issue();
            } else {
                asm volatile("" ::: "memory");
            }
            rows(qnn);
            asm volatile("" ::: "memory");
#pragma unroll
            for (int sI = 0; sI < 2; ++sI)
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    dv[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(td[sI][d], pfr[sI], dv[d], 0, 0, 0);
                    dk[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(tq[sI][d], dsf[sI], dk[d], 0, 0, 0);
                    if (MORE && sI == 0) dk[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(tq[sI][d], low, dk[d], 0, 0, 0);
                }
            s = sn;
            dp = dpn;
        };
        issue();
        settle(kf);
        settle(vf);
        stage_fence();
        issue();  // (the first fence of the walk waits for it)
        rows(smem);
        scores(s, dp, (const float*)(smem + 2 * TILEB));
        rows(smem + BLOCKB);
        int slot = 0, rel = -wave;
        for (int i = 0, it2 = 0; i < steps; ++i) {
            const char* qb = smem + slot * STAGEB;
            const float* stat = (const float*)(qb + 2 * TILEB);
            slot = slot == 2 ? 0 : slot + 1;
            // (behind the last tile: the slot that was read two tiles ago, or nothing yet; its scores are not used)
            const char* qn = smem + slot * STAGEB;
            step(qb, stat, rel, stat + 32, qn, std::true_type{});
            step(qb + BLOCKB, stat + 32, rel + 1, (const float*)(qn + 2 * TILEB), qn + BLOCKB, std::false_type{});
            rel += 2;
            if (++it2 == per_head) { it2 = 0; rel = -wave; }
        }
    }
    if (a.parts > 1) {
        if (!kok) return;
        const long long w = (long long)a.Hkv * D, plane = a.rows * w;
        float* p = a.part + 2 * part * plane + row * w + kvh * D + 4 * hh;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                *(f32x4*)(p + d * 32 + 8 * g) = f32x4{dk[d][4 * g], dk[d][4 * g + 1], dk[d][4 * g + 2], dk[d][4 * g + 3]};
                *(f32x4*)(p + plane + d * 32 + 8 * g) = f32x4{dv[d][4 * g], dv[d][4 * g + 1], dv[d][4 * g + 2], dv[d][4 * g + 3]};
            }
        return;
    }
    store_row<D>(a.dK + row * a.lddk + kvh * D, nullptr, dk, a.scale, hh, kok);
    store_row<D>(a.dV + row * a.lddv + kvh * D, nullptr, dv, 1.0f, hh, kok);
}

template <int D, int W>
__global__ __launch_bounds__(64 * W, D == 64 ? 2 : 1) void packed_bwd_dkv_kernel(const PackedArgs a) {
    __shared__ __attribute__((aligned(1024))) char smem[3 * dkv_stage<D>()];
    Tile tl;
    const int units = a.Hkv * a.parts;
    if (!find_tile<32 * W>(a, blockIdx.x / units, true, tl)) return;
    if (a.parts > 1 && tl.tail) return;  // (packed_join_kernel's)
    dkv_walk<D, W>(a, tl, blockIdx.x % a.Hkv, blockIdx.x % units / a.Hkv, smem);
}

// ------------------------------------------------------------------ backward of short sequences
// A sequence of at most 64 rows fits two waves and its operands one stage: one workgroup takes it, for a key head and the query heads
// of its group in turn, from loads to dQ, dK and dV.  Every operand is read once, S and dP are computed once.  Waves own 32 keys as
// in the dK / dV kernel (block pairs (0, 0), (0, 1); (1, 1)); dS, rounded for dK's product, is also left in LDS as rows of keys, from
// where transposed reads give the B operand of dQ^T = K^T dS^T, the waves owning 32 queries now.
// Sequences that are longer, a few among many, have the launch's first workgroups, which end at once where there are none: a tile of
// 64 rows and a head for dQ by the walk above, or a key head for dK and dV in steps of one stage, delta taken anew.  That is slower
// than the kernels above where one sequence holds most of the rows (3000 and 63 of 9, 16 heads: 151 us against 127, with 4 key heads
// 495 / 251), faster where prompts are prompts (64 of up to 64 rows, 16 heads 15.3 / 22.9; 256 of up to 77: 61 / 92; 4096: 1035 / 1741;
// d 128 29 / 54, 140 / 230, 2207 / 3854).  What sends a batch here is its mean length, in which empty sequences count, and rows behind the
// last one too: 16 sequences of 1000 rows and 300 empty ones take 325 us against 189 without the empty ones, with 4 key heads 408 / 187.
// Bound by the latency of a workgroup's chain of loads and barriers: at 4096 prompts it moves 3.0 TB/s, the matrix pipe busy 0.06 and the
// vector pipe 0.26 of the time, the waves waiting half of theirs; at d 128 one wave a SIMD (426 registers), 2.2 ms.
// W 3: the same for up to 96 rows, where they have more than 64 in the mean (64 x 77 rows, 16 heads 28.5 us against 43 by the kernels above,
// 256 of them 112 / 170; with fewer rows the two waves are faster: 64 of up to 77 rows 18.9 / 23.7).
template <int D, int W>
constexpr int short_smem() {  // Q, dO, K; dS and its low parts (the third block of queries in planes of its own); lse, delta; or what dq_walk needs
    return std::max(3 * 32 * W * 2 * D + (W - 1) * (64 + 16) * 128 + 256 * W, 5 * PA_TILE * 2 * D);
}
// dK and dV of 32 W keys from row k0 of a sequence on; WHOLE: they are all of it, dQ too
template <int D, int W, bool WHOLE>
__device__ __forceinline__ void key_tile(const PackedArgs& a, int start, int len, int k0, bool tail, int kvh, char* smem) {
    constexpr int ROWS = 32 * W;
    constexpr int NK = D / 16, ND = D / 32, ROWB = 2 * D, TILEB = ROWS * ROWB, BLOCKB = 32 * ROWB, SROW = 128;
    char *qs = smem, *dos = smem + TILEB, *ks_ = smem + 2 * TILEB, *dss = smem + 3 * TILEB;
    char* lows = dss + (W - 1) * 64 * SROW;  // what the rounding of dS took away from keys 0 .. 15 and 64 .. 79
    float* stat = (float*)(lows + (W - 1) * 16 * SROW);
    // dS of key block kb and query block b < 2: rows 32 kb + key, half b; of query block 2: rows (kb == 2 ? 32 : 0) + key of the second plane,
    // half kb & 1.  Low parts of kb 0, b < 2: rows key, half b; b 2: rows key of the second plane, half kb / 2.
    auto ds_row = [](int kb, int b) { return b < 2 ? 32 * kb : 64 + (kb == 2 ? 32 : 0); };
    auto ds_half = [](int kb, int b) { return b < 2 ? b : kb & 1; };
    auto low_row = [](int b) { return b < 2 ? 0 : 16; };
    auto low_half = [](int kb, int b) { return b < 2 ? b : kb >> 1; };
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l31 = lane & 31, hh = lane >> 5, G = a.H / a.Hkv, own = wave * 32 + l31;
    const bool ok = k0 + own < len, busy = k0 + wave * 32 < len;
    const long long row = start + (ok ? k0 + own : 0);
    const long long ldqb = a.ldq * 2, lddob = a.lddo * 2, ldkb = a.ldk * 2;
    TileDma<D, W, ROWS> qd, dd, kd;
    qd.init(wave, lane, ldqb);
    dd.init(wave, lane, lddob);
    kd.init(wave, lane, ldkb);
    const unsigned lds0 = lds_addr(smem);
    if constexpr (WHOLE) kd.issue(row_rsrc((const char*)(a.K + (long long)start * a.ldk + kvh * D), len, ldkb, ROWB), lds0 + 2 * TILEB);
    bf16x8 kf[NK], vf[NK];
    load_frags<D>(kf, a.K + row * a.ldk + kvh * D, hh, ok);
    load_frags<D>(vf, a.V + row * a.ldv + kvh * D, hh, ok);
    int rread[NK], tlo[ND], thi[ND];
#pragma unroll
    for (int ks = 0; ks < NK; ++ks) rread[ks] = l31 * ROWB + (((2 * ks + hh) ^ swz<D>(l31)) << 4);
#pragma unroll
    for (int d = 0; d < ND; ++d) tr_lane<D>(lane, d, tlo[d], thi[d]);
    f32x16 dk[ND], dv[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) { dk[d][e] = 0.f; dv[d][e] = 0.f; }
    int g = 0, q0 = k0;  // head of the group, first row of the tile of queries
    for (bool first = true; g < (tail ? 0 : G); first = false) {
        const int h = kvh * G + g, left = min(len - q0, ROWS);
        const bool qok = WHOLE ? ok : own < left;
        const long long qrow = WHOLE ? row : start + q0 + (qok ? own : 0);
        if (!first) __syncthreads();
        qd.issue(row_rsrc((const char*)(a.Q + (long long)(start + q0) * a.ldq + h * D), left, ldqb, ROWB), lds0);
        dd.issue(row_rsrc((const char*)(a.dO + (long long)(start + q0) * a.lddo + h * D), left, lddob, ROWB), lds0 + TILEB);
        // delta of the wave's 32 queries: O and what its rounding took away from memory, dO from LDS
        u32x4 ov[NK], lv[NK];
#pragma unroll
        for (int ks = 0; ks < NK; ++ks) {
            ov[ks] = lv[ks] = u32x4{0u, 0u, 0u, 0u};
            if (qok) ov[ks] = *(const u32x4*)(a.O + qrow * a.ldo + h * D + ks * 16 + hh * 8);
            if (qok && a.o_low) lv[ks] = *(const u32x4*)(a.o_low + (qrow * a.H + h) * D + ks * 16 + hh * 8);
        }
        const float lse = qok ? a.lse[(long long)h * a.rows + qrow] : 0.f;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the wave's own pieces; the other's behind the barrier)
        __syncthreads();
        float dlt = 0.f;
#pragma unroll
        for (int ks = 0; ks < NK; ++ks) {
            float x[8], l[8], y[8];
            unpack8(ov[ks], x);
            unpack8(lv[ks], l);
            unpack8(*(const u32x4*)(dos + wave * BLOCKB + rread[ks]), y);
#pragma unroll
            for (int j = 0; j < 8; ++j) dlt = fmaf(x[j] + l[j], y[j], dlt);
        }
        dlt = half_sum(dlt);
        if (hh == 0) {  // (queries behind the end: zero, P = 1 meets only zeros)
            stat[own] = lse;
            stat[ROWS + own] = -dlt;
        }
        __syncthreads();
        if (busy) {
#pragma nounroll
            for (int b = WHOLE || q0 == k0 ? wave : 0; b < W && b * 32 < left; ++b) {
                const float* st = stat + 32 * b;
                const char *qb = qs + b * BLOCKB, *db = dos + b * BLOCKB;
                f32x16 s, dp;
#pragma unroll
                for (int gq = 0; gq < 4; ++gq) {
                    const f32x4 d4 = *(const f32x4*)(st + ROWS + 8 * gq + 4 * hh);
#pragma unroll
                    for (int j = 0; j < 4; ++j) { s[4 * gq + j] = 0.f; dp[4 * gq + j] = FROM_DELTA<D> ? d4[j] : 0.f; }
                }
#pragma unroll
                for (int ks = 0; ks < NK; ++ks) {
                    s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(qb + rread[ks]), kf[ks], s, 0, 0, 0);
                    dp = __builtin_amdgcn_mfma_f32_32x32x16_bf16(*(const bf16x8*)(db + rread[ks]), vf[ks], dp, 0, 0, 0);
                }
                if constexpr (!FROM_DELTA<D>) add_delta(dp, st + ROWS, hh);
                if (b == wave && (WHOLE || q0 == k0)) {
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if ((e & 3) + 8 * (e >> 2) + 4 * hh < l31) s[e] = -INFINITY;  // P = 0, dS = 0
                    if (q0 + b + hh == 0) dp[0] = 0.f;                                // (query 0 sees one key: P = 1, dS = 0)
                }
                bf16x8 pfr[2], dsf[2], low0;
#pragma unroll
                for (int sI = 0; sI < 2; ++sI) {
                    float p[8], ds[8];
#pragma unroll
                    for (int gq = 0; gq < 2; ++gq) {
                        const f32x4 l4 = *(const f32x4*)(st + 16 * sI + 8 * gq + 4 * hh);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int e = 8 * sI + 4 * gq + j;
                            p[4 * gq + j] = __builtin_amdgcn_exp2f(fmaf(s[e], a.scale_log2e, -l4[j]));
                            ds[4 * gq + j] = p[4 * gq + j] * dp[e];
                        }
                    }
                    pfr[sI] = __builtin_bit_cast(bf16x8, pack8(p));
                    const u32x4 packed = pack8(ds);
                    dsf[sI] = __builtin_bit_cast(bf16x8, packed);
                    const u32x4 low = rounded_off(ds, packed);
                    if (sI == 0) low0 = __builtin_bit_cast(bf16x8, low);
                    if constexpr (WHOLE) {  // queries 32 b + 16 sI + 8 gq + 4 hh .. + 3 of the lane's key
                        char* to = dss + (ds_row(wave, b) + l31) * SROW;
                        char* lo = lows + (low_row(b) + l31) * SROW;
#pragma unroll
                        for (int gq = 0; gq < 2; ++gq) {
                            const int c = 2 * sI + gq, x = swz<64>(l31);
                            *(u32x2*)(to + (((4 * ds_half(wave, b) + c) ^ x) << 4) + 8 * hh) = u32x2{packed[2 * gq], packed[2 * gq + 1]};
                            if (!(wave & 1) && l31 < 16)
                                *(u32x2*)(lo + (((4 * low_half(wave, b) + c) ^ x) << 4) + 8 * hh) = u32x2{low[2 * gq], low[2 * gq + 1]};
                        }
                    }
                }
#pragma unroll
                for (int sI = 0; sI < 2; ++sI)
#pragma unroll
                    for (int d = 0; d < ND; ++d) {
                        const char *x = qb + sI * 16 * ROWB, *y = db + sI * 16 * ROWB;
                        dv[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(tr_pair(y + tlo[d], y + thi[d]), pfr[sI], dv[d], 0, 0, 0);
                        const bf16x8 qt = tr_pair(x + tlo[d], x + thi[d]);
                        dk[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qt, dsf[sI], dk[d], 0, 0, 0);
                        if (!(b & 1) && sI == 0) dk[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(qt, low0, dk[d], 0, 0, 0);
                    }
            }
        }
        if (!WHOLE && q0 + PA_TILE < len) {
            q0 += PA_TILE;
            continue;
        }
        q0 = k0;
        ++g;
        if constexpr (!WHOLE) continue;
        __syncthreads();
        if (busy) {
            f32x16 dq[ND];
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) dq[d][e] = 0.f;
            for (int b = 0; b <= wave; ++b) {
                int qlo, qhi, llo, lhi;
                tr_lane<64>(lane, ds_half(b, wave), qlo, qhi);
                tr_lane<64>(lane, low_half(b, wave), llo, lhi);
                const char* lw = lows + low_row(wave) * SROW;
#pragma unroll
                for (int sI = 0; sI < 2; ++sI) {
                    const char *x = dss + (ds_row(b, wave) + 16 * sI) * SROW, *y = ks_ + b * BLOCKB + sI * 16 * ROWB;
                    const bf16x8 f = tr_pair(x + qlo, x + qhi);
#pragma unroll
                    for (int d = 0; d < ND; ++d) {
                        const bf16x8 kt = tr_pair(y + tlo[d], y + thi[d]);
                        dq[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kt, f, dq[d], 0, 0, 0);
                        if (!(b & 1) && sI == 0) dq[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kt, tr_pair(lw + llo, lw + lhi), dq[d], 0, 0, 0);
                    }
                }
            }
            store_row<D>(a.dQ + row * a.lddq + h * D, nullptr, dq, a.scale, hh, ok);
        }
    }
    if (busy) {
        store_row<D>(a.dK + row * a.lddk + kvh * D, nullptr, dk, a.scale, hh, ok);
        store_row<D>(a.dV + row * a.lddv + kvh * D, nullptr, dv, 1.0f, hh, ok);
    }
}
template <int D, int W>
__global__ __launch_bounds__(64 * W, D == 64 ? 2 : 1) void packed_bwd_short_kernel(const PackedArgs a) {
    __shared__ __attribute__((aligned(1024))) char smem[short_smem<D, W>()];
    const int at = (int)blockIdx.x - a.rest;
    if (at >= 0) {
        const int i = at / a.Hkv, start = min(max(a.cu[i], 0), a.rows), len = min(max(a.cu[i + 1], start), a.rows) - start;
        if (len > 0 && len <= a.skip) key_tile<D, W, true>(a, start, len, 0, false, at % a.Hkv, smem);
        return;
    }
    if (threadIdx.x >= 128) return;  // (a tile of 64 rows: two waves; barriers wait for those that are left)
    const int u = blockIdx.x, groups = (a.H + a.Hkv + a.per - 1) / a.per, u0 = u % groups;
    Tile tl;
    if (!find_tile<PA_TILE>(a, u / groups, false, tl)) return;
    for (int j = u0; j < a.H + a.Hkv; j += groups) {
        if (j > u0) __syncthreads();
        // (one unit a workgroup: the longest walks come first, dQ's of the last tile and dK's of the first; more: their lengths add up
        // to the same for every tile)
        if (j < a.Hkv) key_tile<D, 2, false>(a, tl.start, tl.len, (a.per == 1 ? tl.ntiles - 1 - tl.tile : tl.tile) * PA_TILE, tl.tail, j, smem);
        else dq_walk<D, 2>(a, tl, j - a.Hkv, smem);
    }
}

// dK and dV of the parts, in their order: a thread per 8 channels of a row and gradient.  Bound by memory: 2 parts of 13.6k rows x 256,
// 56 MB read and 14 written, 12.5 us = 5.6 TB/s.
__global__ __launch_bounds__(256) void packed_join_kernel(const PackedArgs a, int width) {
    const int end = min(max(a.cu[a.n_seq], 0), a.rows), chunks = width / 8;
    const long long plane = (long long)a.rows * width, n = 2ll * a.rows * chunks;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        const int c = (int)(i % chunks) * 8, which = (int)(i / chunks & 1);
        const long long row = i / chunks >> 1;
        float s[8] = {};
        if (row < end) {
            const float* p = a.part + which * plane + row * width + c;
            for (int k = 0; k < a.parts; ++k, p += 2 * plane) {
                const f32x4 x = *(const f32x4*)p, y = *(const f32x4*)(p + 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) { s[e] += x[e]; s[4 + e] += y[e]; }
            }
        } else if (!a.zero_tail) continue;
        if (which == 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] *= a.scale;
        }
        *(u32x4*)((which ? a.dV + row * a.lddv : a.dK + row * a.lddk) + c) = pack8(s);
    }
}

// the most tiles of `step` rows that n_seq sequences (and the rows behind them) can have in `rows` rows, or their places
long long most_tiles(int rows, int n_seq, int step, int tail) {
    if (n_seq > FEW_SEQS) return (long long)rows / step + n_seq + tail;
    return ((long long)rows + (long long)(n_seq + tail) * (step - 1)) / step;
}

// Whether most sequences fit 64 rows, as far as their mean says.
bool mostly_short(int rows, int n_seq) { return rows <= 64ll * n_seq; }
// What the backward of a batch of prompts takes in one piece: sequences of up to 64 or 96 rows; 0: no such batch.
int short_rows_of(int rows, int n_seq) { return mostly_short(rows, n_seq) ? 64 : rows <= 96ll * n_seq ? 96 : 0; }
// With at most 64 rows the forward has two waves to a workgroup instead of four (d 64; d 128 gains nothing): tiles of 64 rows, where most of
// 128 would have no queries, and four workgroups a CU (as many as their LDS allows) instead of three (64 x 40 rows, 16 heads: 11.0 -> 8.4 us;
// from 77 rows on there is nothing in it).  A wave does the same in both, so a sequence's bits do not show which it was.
int waves_of(int rows, int n_seq, int d) { return d == 64 && mostly_short(rows, n_seq) ? 2 : 4; }

// Into how many parts the walk of a key tile over its group's query heads is cut.  One workgroup walks G heads x the queries
// behind its keys; with few key heads and long sequences the longest of those walks outlasts the rest of the grid.  Parts cost
// fp32 sums through memory (16 bytes a channel), so only walks of at least 8 tiles a head on average are cut, and only while the
// grid has fewer than 768 workgroups (three a CU).  The order of a group's sum, and with it the last bits of dK and dV, follows from the
// number of parts.
int parts_of(int n_seq, int rows, int H, int Hkv) {
    const int G = H / Hkv;
    if (rows < 512ll * (n_seq > 0 ? n_seq : 1)) return 1;
    int p = 1;
    while (p < G && most_tiles(rows, n_seq, 128, 0) * Hkv * p < 768) {
        do ++p;
        while (G % p);
    }
    return p;
}
size_t delta_bytes(int rows, int H) { return ((size_t)rows * H * 4 + 255) & ~(size_t)255; }

// Workgroups for sequences that are longer than most, of which there may be none: so many at most, each with several heads if need
// be (prompts of up to 77 rows, 8 heads, backward: 512 of them 56 us with 4096, 61 with 8192, 71 with 16384; 1024 and one sequence of 4096
// rows 667 / 470 / 316); fewer where the kernel has fewer workgroups a CU (64 x 77 rows, 16 heads 28.5 us with 2048, 32 with 8192)
long long most_empty(int d, int short_rows) { return d == 64 && short_rows == 64 ? 8192 : 2048; }
constexpr long long MOST_GROUPS = (1 << 24) - 1;  // (a launch has less than 2^32 threads)

RowSpan offsets(const int32_t* cu, int n_seq) { return {cu, 4 * (n_seq + 1ll), 4 * (n_seq + 1ll), 1}; }
RowSpan span(const void* p, int ld, int width, int rows) { return {p, 2ll * ld, 2ll * width, rows}; }
bool row_ok(const void* p, int ld, long long width) { return p && !((uintptr_t)p & 15) && !(ld & 7) && ld >= width; }

}  // namespace

extern "C" int ccnet_attention_packed_bf16(const void* Q, int ldq, const void* K, int ldk, const void* V, int ldv, void* O, int ldo,
                                           const int32_t* cu_seqlens, int n_seq, int rows, int H, int Hkv, int d, float scale,
                                           int zero_tail, float* lse, void* o_low, void* stream) {
    if (rows < 0 || n_seq < 0 || H <= 0 || Hkv <= 0 || H % Hkv || !(scale > 0.f) || scale > 3.0e38f) return CCNET_EINVAL;
    if ((d != 64 && d != 128) || rows > (1 << 29) || H > (1 << 20)) return CCNET_EUNSUP;
    if (rows == 0) return CCNET_OK;
    if (!cu_seqlens || !row_ok(Q, ldq, H * d) || !row_ok(K, ldk, Hkv * d) || !row_ok(V, ldv, Hkv * d) || !row_ok(O, ldo, H * d)) return CCNET_EINVAL;
    if (((uintptr_t)o_low & 15) || ((uintptr_t)lse & 3) || ((uintptr_t)cu_seqlens & 3)) return CCNET_EINVAL;
    if (ldk > (1 << 24) || ldv > (1 << 24)) return CCNET_EUNSUP;
    const RowSpan q = span(Q, ldq, H * d, rows), k = span(K, ldk, Hkv * d, rows), v = span(V, ldv, Hkv * d, rows), o = span(O, ldo, H * d, rows),
                  low = span(o_low, H * d, H * d, rows), stat = span(lse, 2 * rows, 2 * rows, H);
    if (!spans_apart(o, k) || !spans_apart(o, v) || !(spans_apart(o, q) || (O == Q && ldo == ldq))) return CCNET_EINVAL;
    if (!spans_apart(low, q) || !spans_apart(low, k) || !spans_apart(low, v) || !spans_apart(low, o)) return CCNET_EINVAL;
    for (const RowSpan& s : {q, k, v, o, low})
        if (!spans_apart(stat, s)) return CCNET_EINVAL;
    PackedArgs a{};
    a.Q = (const __bf16*)Q; a.K = (const __bf16*)K; a.V = (const __bf16*)V; a.out = (__bf16*)O;
    a.ldq = ldq; a.ldk = ldk; a.ldv = ldv; a.ldo = ldo;
    a.cu = cu_seqlens; a.n_seq = n_seq; a.rows = rows; a.H = H; a.Hkv = Hkv;
    a.scale = scale; a.scale_log2e = scale * 1.4426950408889634f; a.zero_tail = zero_tail != 0; a.lse = lse;
    a.o_low = (__bf16*)o_low;
    // 64 queries a wave (a K or V fragment feeds two products) where whole 256-query tiles are the rule and there are at least four of
    // them a CU: 64 x 1024 rows, 16 heads 231 us against 255, 4 x 8192 rows, 32 heads 1160 / 1236; with fewer the longest walks
    // outlast the rest (2048 rows, 16 heads 47 / 31), with shorter sequences the last tiles are mostly empty (300 x 300 rows 381 / 371).
    // Both blocks' running maxima move together, so that P, and o and lse in their last bits, may round differently than in the narrow form.
    const bool wide = d == 64 && rows >= 512ll * n_seq && (long long)rows * H >= 256ll * 1024;
    const int waves = waves_of(rows, n_seq, d);
    const long long grid = most_tiles(rows, n_seq, wide ? 256 : 32 * waves, a.zero_tail) * H;
    if (grid > MOST_GROUPS) return CCNET_EUNSUP;
    for (const RowSpan& s : {o, low, stat})
        if (!spans_apart(offsets(cu_seqlens, n_seq), s)) return CCNET_EINVAL;
    if (grid == 0) return CCNET_OK;
    hipStream_t st = (hipStream_t)stream;
    const dim3 g((unsigned)grid), b(64 * waves);
    if (wide) hipLaunchKernelGGL((packed_fwd_kernel<64, 2, 4>), g, dim3(256), 0, st, a);
    else if (d == 128) hipLaunchKernelGGL((packed_fwd_kernel<128, 1, 4>), g, b, 0, st, a);
    else if (waves == 4) hipLaunchKernelGGL((packed_fwd_kernel<64, 1, 4>), g, b, 0, st, a);
    else hipLaunchKernelGGL((packed_fwd_kernel<64, 1, 2>), g, b, 0, st, a);
    CCNET_LAUNCH_CHECK();
    return CCNET_OK;
}

extern "C" size_t ccnet_attention_packed_bwd_workspace_bytes(int n_seq, int rows, int H, int Hkv, int d) {
    if (rows <= 0 || n_seq < 0 || H <= 0 || Hkv <= 0 || H % Hkv || (d != 64 && d != 128)) return 0;
    const int parts = parts_of(n_seq, rows, H, Hkv);
    return delta_bytes(rows, H) + (parts > 1 ? (size_t)parts * 2 * rows * Hkv * d * 4 : 0);
}

extern "C" int ccnet_attention_packed_bwd_bf16(const void* Q, int ldq, const void* K, int ldk, const void* V, int ldv, const void* O,
                                               int ldo, const void* o_low, const void* dO, int lddo, const float* lse, void* dQ, int lddq,
                                               void* dK, int lddk, void* dV, int lddv, const int32_t* cu_seqlens, int n_seq, int rows,
                                               int H, int Hkv, int d, float scale, int zero_tail, void* workspace, size_t workspace_bytes,
                                               void* stream) {
    if (rows < 0 || n_seq < 0 || H <= 0 || Hkv <= 0 || H % Hkv || !(scale > 0.f) || scale > 3.0e38f) return CCNET_EINVAL;
    if ((d != 64 && d != 128) || rows > (1 << 29) || H > (1 << 20)) return CCNET_EUNSUP;
    if (rows == 0) return CCNET_OK;
    if (!cu_seqlens || !lse || !workspace || ((uintptr_t)workspace & 15) || ((uintptr_t)o_low & 15) || !row_ok(Q, ldq, H * d) ||
        !row_ok(K, ldk, Hkv * d) || !row_ok(V, ldv, Hkv * d) || !row_ok(O, ldo, H * d) || !row_ok(dO, lddo, H * d) ||
        !row_ok(dQ, lddq, H * d) || !row_ok(dK, lddk, Hkv * d) || !row_ok(dV, lddv, Hkv * d))
        return CCNET_EINVAL;
    if (((uintptr_t)lse & 3) || ((uintptr_t)cu_seqlens & 3)) return CCNET_EINVAL;
    if (ldq > (1 << 24) || ldk > (1 << 24) || ldv > (1 << 24) || lddo > (1 << 24)) return CCNET_EUNSUP;
    const size_t need = ccnet_attention_packed_bwd_workspace_bytes(n_seq, rows, H, Hkv, d);
    if (workspace_bytes < need) return CCNET_EWS;
    const RowSpan in[] = {span(Q, ldq, H * d, rows),         span(K, ldk, Hkv * d, rows),  span(V, ldv, Hkv * d, rows),
                          span(O, ldo, H * d, rows),         span(dO, lddo, H * d, rows),  span(o_low, H * d, H * d, rows),
                          span(lse, 2 * rows, 2 * rows, H)};
    const RowSpan out[] = {span(dQ, lddq, H * d, rows), span(dK, lddk, Hkv * d, rows), span(dV, lddv, Hkv * d, rows)};
    const RowSpan ws{workspace, (long long)need, (long long)need, 1};
    for (const RowSpan& s : in)
        if (!spans_apart(ws, s)) return CCNET_EINVAL;
    for (int i = 0; i < 3; ++i) {
        if (!spans_apart(ws, out[i])) return CCNET_EINVAL;
        for (const RowSpan& s : in)
            if (!spans_apart(out[i], s)) return CCNET_EINVAL;
        for (int j = 0; j < i; ++j)
            if (!spans_apart(out[i], out[j])) return CCNET_EINVAL;
    }
    PackedArgs a{};
    a.Q = (const __bf16*)Q; a.K = (const __bf16*)K; a.V = (const __bf16*)V; a.O = (const __bf16*)O; a.dO = (const __bf16*)dO;
    a.o_low = (__bf16*)o_low;
    a.dQ = (__bf16*)dQ; a.dK = (__bf16*)dK; a.dV = (__bf16*)dV;
    a.ldq = ldq; a.ldk = ldk; a.ldv = ldv; a.ldo = ldo; a.lddo = lddo; a.lddq = lddq; a.lddk = lddk; a.lddv = lddv;
    a.cu = cu_seqlens; a.n_seq = n_seq; a.rows = rows; a.H = H; a.Hkv = Hkv;
    a.scale = scale; a.scale_log2e = scale * 1.4426950408889634f; a.zero_tail = zero_tail != 0;
    a.lse = (float*)lse;
    a.delta = (float*)workspace;
    a.part = (float*)((char*)workspace + delta_bytes(rows, H));
    a.parts = parts_of(n_seq, rows, H, Hkv);
    const int short_rows = short_rows_of(rows, n_seq);
    const long long tiles = most_tiles(rows, n_seq, 128, a.zero_tail), qtiles = most_tiles(rows, n_seq, short_rows ? PA_TILE : 128, a.zero_tail);
    if (qtiles * H > MOST_GROUPS) return CCNET_EUNSUP;
    for (const RowSpan& s : {out[0], out[1], out[2], ws})
        if (!spans_apart(offsets(cu_seqlens, n_seq), s)) return CCNET_EINVAL;
    if (tiles == 0 && qtiles == 0) return CCNET_OK;
    hipStream_t st = (hipStream_t)stream;
    if (short_rows) {
        a.skip = short_rows;
        long long longer = qtiles;  // tiles of sequences of more rows than that, or the rows behind the last
        if (n_seq <= FEW_SEQS) longer = std::min(longer, (long long)rows / PA_TILE + rows / (short_rows + 1) + 1);
        const long long most = most_empty(d, short_rows);
        a.per = (int)((longer * (H + Hkv) + most - 1) / most);
        const long long rest = longer * ((H + Hkv + a.per - 1) / a.per), groups = (long long)n_seq * Hkv + rest;
        a.rest = (int)rest;
        if (groups > MOST_GROUPS) return CCNET_EUNSUP;
        const dim3 gs((unsigned)groups);
        if (d == 128 && short_rows == 96) hipLaunchKernelGGL((packed_bwd_short_kernel<128, 3>), gs, dim3(192), 0, st, a);
        else if (d == 128) hipLaunchKernelGGL((packed_bwd_short_kernel<128, 2>), gs, dim3(128), 0, st, a);
        else if (short_rows == 96) hipLaunchKernelGGL((packed_bwd_short_kernel<64, 3>), gs, dim3(192), 0, st, a);
        else hipLaunchKernelGGL((packed_bwd_short_kernel<64, 2>), gs, dim3(128), 0, st, a);
        CCNET_LAUNCH_CHECK();
        return CCNET_OK;
    }
    const dim3 gq((unsigned)(qtiles * H)), gk((unsigned)(tiles * Hkv * a.parts));
    if (d == 128) hipLaunchKernelGGL((packed_bwd_dq_kernel<128, 4>), gq, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((packed_bwd_dq_kernel<64, 4>), gq, dim3(256), 0, st, a);
    CCNET_LAUNCH_CHECK();
    if (tiles == 0) return CCNET_OK;
    if (d == 128) hipLaunchKernelGGL((packed_bwd_dkv_kernel<128, 4>), gk, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((packed_bwd_dkv_kernel<64, 4>), gk, dim3(256), 0, st, a);
    CCNET_LAUNCH_CHECK();
    if (a.parts > 1) {
        const long long threads = 2ll * rows * (Hkv * d / 8);
        hipLaunchKernelGGL(packed_join_kernel, dim3((unsigned)std::min<long long>((threads + 255) / 256, 1 << 20)), dim3(256), 0, st, a, Hkv * d);
        CCNET_LAUNCH_CHECK();
    }
    return CCNET_OK;
}
