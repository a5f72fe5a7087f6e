// Selective state space scan over packed requests, with the requests' states in
// a pool of slots.  With delta = softplus(dt + bias), channel d's N states and
// output are
//   h[n] = exp(delta A[d][n]) h[n] + delta x B[n],   y = (sum_n h[n] C[n] + D x) silu(z).
//
// Bound by the exponential unit: N exponentials a row and channel, two for
// delta and two for the gate, at 16 a clock and multiprocessor.  So everything
// else is kept small beside them.  K lanes share a channel and hold SPT of its
// states each in registers; a channel's delta, gate and output are its lanes'
// own work (of four rows, each lane has its part of them), and only B and C,
// which all channels of a group read, go through shared memory, where a block
// converts them once for its 128 / K channels.  The multiply-adds are packed in
// pairs of states.
//
// A request is walked row by row; walking requests in pieces at once costs twice
// the work (a first walk finds each piece's own state and sum of delta, a short
// kernel carries the states from piece to piece, and the last walk starts from
// them), so that only a request of more than its share is split: a piece has the
// rows that give the device one wave of blocks, and a request of up to five of
// them is walked alone (one prompt of 4000 rows, bfloat16, in pieces and alone:
// 5120 channels, 14 pieces, 247 and 720 us; 12,000, six, 548 and 725; 16,384, four,
// 809 and 770).
//
// Measured (N = 16): 64 prompts of 0 to 511 rows x 5120 bfloat16 channels 480 us --
// 20 exponentials a row and channel would be 372 us, and a walk of the same
// instructions without its inputs takes 168 cycles for 32 channels, 387 us -- and
// 8192 rows x 1536 half channels in 49 pieces 157 us (apart and cold: the first walk
// 76, the carry 10, the last walk 84; their exponentials 50 and 55).  A polynomial in
// place of an eighth of the exponentials takes as long (167 cycles), of a quarter
// longer (177).
#pragma once
#include <limits.h>

#include <type_traits>

#include "kernels.h"
#include "paged.h"
#include "recurrent.cuh"

namespace krk {
namespace {

constexpr int CARRY_AHEAD = 16;
constexpr int SCAN_GROUP = 4;  // rows whose outputs are formed together

// K lanes share a channel of N <= K * SPT states.
template <typename T, int K, int SPT, bool AHEAD>
struct ScanShape {
    static constexpr int CH = SCAN_THREADS / K, NP = K * SPT;
    static constexpr int MOST = AHEAD ? (sizeof(T) == 2 ? 16 : 8) : 32;
    static constexpr int ROWS = NP * MOST <= 1024 ? MOST : 1024 / NP;  // a tile
    static constexpr int BC = 2 * ROWS * NP;                           // elements of B and C in it
    static constexpr int F = (BC + SCAN_THREADS - 1) / SCAN_THREADS;   // and those that a thread stages
    static constexpr int OWN = K < SCAN_GROUP ? SCAN_GROUP / K : 1;    // rows of a group whose inputs are a lane's work
    static constexpr int SHARE = K < SCAN_GROUP ? 1 : K / SCAN_GROUP;  // lanes that have the same ones
};

// How a request is split.
struct ScanSplit {
    int rows;       // a piece's
    float* start;   // [pieces of split requests][D][N]: the states that pieces start from
    float* sum;     // [pieces of split requests][D]: their sums of delta
    int room;       // pieces of split requests that there is room for: more come from offsets that do not ascend,
                    // and the requests that have none are left alone
};
KRK_DEV int scan_pieces(int n, int rows) { return rows > 0 && n > (int64_t)SCAN_ALONE * rows ? (n - 1) / rows + 1 : 1; }

// The piece-th piece of the requests that are split: its request, its place
// there, and the place of the request's first one among all; FIRST: the piece-th
// such request's first piece.  request < 0: there are not so many.
struct ScanPiece {
    int request, at, first;
};
template <bool FIRST>
KRK_DEV ScanPiece find_piece(const int32_t* cu, int S, int T, int rows, int piece) {
    __shared__ int warp_sum[2][SCAN_THREADS / 32];
    __shared__ ScanPiece found;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    int before = 0, places = 0;  // of the requests so far: what is counted, and their pieces
    if (tid == 0) found.request = -1;
    __syncthreads();
    for (int s0 = 0; s0 < S; s0 += SCAN_THREADS) {
        const int s = s0 + tid;
        int m = 0;
        if (s < S) {
            m = scan_pieces(clamp_row(cu[s + 1], T) - clamp_row(cu[s], T), rows);
            if (m == 1) m = 0;
        }
        const int n = FIRST ? m > 0 : m;
        int x = n, y = m;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int p = __shfl_up_sync(0xffffffffu, x, o), q = __shfl_up_sync(0xffffffffu, y, o);
            if (lane >= o) x += p, y += q;
        }
        if (lane == 31) warp_sum[0][warp] = x, warp_sum[1][warp] = y;
        __syncthreads();
        int all = 0, all_places = 0;
#pragma unroll
        for (int w = 0; w < SCAN_THREADS / 32; ++w) {
            if (w == warp) x += all, y += all_places;
            all += warp_sum[0][w];
            all_places += warp_sum[1][w];
        }
        const int at = piece - before - (x - n);
        if (at >= 0 && at < n) found = {s, at, places + y - m};
        before += all;
        places += all_places;
        __syncthreads();
        if (found.request >= 0) break;
    }
    return found;
}

// The turn-th unit of work of the last walk -- a request, or a piece of one that
// is split -- of up to S + room.  The longest ones come first, so that what is
// left when most blocks have ended is short; of more requests than a block has
// threads, the pieces come first, then the requests in their order.
KRK_DEV ScanPiece find_unit(const int32_t* cu, int S, int T, const ScanSplit& split, int turn) {
    if (S > SCAN_THREADS) {
        if (turn < split.room) return find_piece<false>(cu, S, T, split.rows, turn);
        const int s = turn - split.room, n = clamp_row(cu[s + 1], T) - clamp_row(cu[s], T);
        return {scan_pieces(n, split.rows) > 1 ? -1 : s, 0, 0};
    }
    __shared__ int rows[SCAN_THREADS], pieces[SCAN_THREADS];
    __shared__ ScanPiece found;
    const int s = threadIdx.x;
    const int n = s < S ? clamp_row(cu[s + 1], T) - clamp_row(cu[s], T) : INT_MIN, p = s < S ? scan_pieces(n, split.rows) : 0;
    rows[s] = p > 1 ? split.rows : n;
    pieces[s] = p;
    if (s == 0) found.request = -1;
    __syncthreads();
    // the units before this request's, and the pieces of split requests with a lower number
    int before = 0, first = 0;
    for (int i = 0; i < S; ++i) {
        const bool sooner = rows[i] > rows[s] || (rows[i] == rows[s] && i < s);
        before += sooner ? pieces[i] : 0;
        first += i < s && pieces[i] > 1 ? pieces[i] : 0;
    }
    if (turn >= before && turn < before + p) found = {s, turn - before, first};
    __syncthreads();
    return found;
}

// Sums each of v's rows over K lanes.  While a lane holds several rows it keeps
// half of them and gives the others away: with K < R lane i ends with rows
// i * R / K .. of the R, else lanes i * K / R .. with row i.
template <int R, int K>
KRK_DEV void sum_rows(float (&v)[R], int lane) {
    int n = R / 2;
#pragma unroll
    for (int off = K / 2; off > 0; off /= 2) {
        if (n > 0) {
            const bool upper = lane & off;
#pragma unroll
            for (int i = 0; i < R / 2; ++i)
                if (i < n) {
                    const float mine = upper ? v[i + n] : v[i], theirs = upper ? v[i] : v[i + n];
                    v[i] = mine + __shfl_xor_sync(0xffffffffu, theirs, off);
                }
            n /= 2;
        } else {
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], off);
        }
    }
}

// Copies 16 bytes, or zeros if there are none, into shared memory.
KRK_DEV void copy16(void* smem, const void* gmem, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(smem)), "l"(gmem), "r"(there ? 16 : 0)
                 : "memory");
}

// What a lane holds besides states: nothing, whole groups of four, or parts of them.
enum ScanPadding { PAD_NONE, PAD_FOURS, PAD_STATES };

// CARRY: the first walk of split requests, which leaves each piece's state from
// zeros, for the piece behind it, and its sum of delta.  AHEAD: x, dt and z, whose
// rows are aligned to 16 bytes, come tile by tile through shared memory, the next
// tile while one is computed; else each lane loads its own, a group ahead.
template <typename T, int K, int SPT, ScanPadding PADDED, bool CARRY, bool AHEAD>
__global__ void __launch_bounds__(SCAN_THREADS, SCAN_BLOCKS) scan_kernel(ScanArgs a, ScanSplit split, int side) {
    using Sh = ScanShape<T, K, SPT, AHEAD>;
    constexpr int CH = Sh::CH, NP = Sh::NP, ROWS = Sh::ROWS, BC = Sh::BC, F = Sh::F, OWN = Sh::OWN,
                  U = SCAN_GROUP;
    constexpr int INPUTS = CARRY ? 2 : 3;
    __shared__ __align__(16) float s_bc[2][ROWS][2][NP];
    __shared__ __align__(16) T s_in[AHEAD ? 2 : 1][INPUTS][AHEAD ? ROWS : 1][AHEAD ? CH : 1];

    const int tid = threadIdx.x, lane = tid % K, per = a.D / a.G;
    const int block = blockIdx.x / side, cb = blockIdx.x - block * side, sides = side / a.G;
    const int g = cb / sides, ch0 = (cb - g * sides) * CH, ch = ch0 + tid / K;  // within the group
    const bool open = ch < per;
    const int d = g * per + (open ? ch : 0);
    const ScanPiece piece = CARRY ? find_piece<false>(a.cu, a.S, a.T, split.rows, block)
                                  : find_unit(a.cu, a.S, a.T, split, block);
    if (piece.request < 0) return;
    const Span span = request_rows(a.cu, piece.request, a.T);
    int to, from;
    if (!request_slots(a.slot, piece.request, to, from)) return;
    const int pieces = scan_pieces(span.end - span.begin, split.rows);
    const bool last = piece.at == pieces - 1;
    if (pieces > 1 && (piece.first < 0 || piece.first > split.room - pieces)) return;
    if (CARRY && last) return;
    const int begin = span.begin + piece.at * split.rows, end = last ? span.end : begin + split.rows;

    // States 4 (q K + lane) .. + 3 of the channel for q < SPT / 4: lanes read B and C side by side.
    const auto state_of = [&](int j) { return 4 * (j / 4 * K + lane) + j % 4; };
    // a lane's groups of four that are there, and the one of them, if any, that holds the last states and others
    const int fours = PADDED ? max(0, (a.N + 3) / 4 - lane + K - 1) / K : SPT / 4;
    const int edge = PADDED == PAD_STATES && a.N / 4 % K == lane ? a.N / 4 / K : -1;
    float2 h[SPT / 2], rate[SPT / 2];
    {
        const float* old = CARRY ? nullptr
                           : pieces > 1 ? split.start + (int64_t)(piece.first + piece.at) * a.D * a.N
                           : from >= 0 ? (const float*)a.slot.state + from * a.slot.stride : nullptr;
#pragma unroll
        for (int j = 0; j < SPT; ++j) {
            const int n = state_of(j);
            const bool in = open && (!PADDED || n < a.N);
            const int64_t at = (int64_t)d * a.N + n;
            const float r = in ? scan_rate(a.a[at]) : 0.0f, v = in && old ? old[at] : 0.0f;
            (j % 2 ? rate[j / 2].y : rate[j / 2].x) = r;
            (j % 2 ? h[j / 2].y : h[j / 2].x) = v;
        }
    }
    const float bias = a.dt_bias ? a.dt_bias[d] : 0.0f, skip = !CARRY && a.d ? a.d[d] : 0.0f;
    const T* bp = (const T*)a.b + g * a.b_sg;
    const T* cp = (const T*)a.c + g * a.c_sg;
    const T zero = from_f32<T>(0.0f);
    const bool gated = !CARRY && a.z;

    // A lane's rows of a group, on their way while the group before is computed; WHOLE: all four rows are there.
    const int own = lane / Sh::SHARE * OWN;
    const T* xp = (const T*)a.x + (begin + own) * a.x_st + d;
    const T* dtp = (const T*)a.dt + (begin + own) * a.dt_st + d;
    const int64_t z_st = gated ? a.z_st : a.x_st;  // (x in place of a gate that there is none of)
    const T* zp = (gated ? (const T*)a.z : (const T*)a.x) + (begin + own) * z_st + d;
    T* outp = (T*)a.out + (begin + own) * a.o_st + d;
    T xr[OWN], dtr[OWN], zr[OWN];
    const auto fetch = [&](int t, auto whole) {
        if constexpr (!AHEAD) {
#pragma unroll
            for (int o = 0; o < OWN; ++o) {
                const bool in = decltype(whole)::value || t + own + o < end;
                xr[o] = in ? *xp : zero;
                dtr[o] = in ? *dtp : zero;
                if (!CARRY) zr[o] = in ? *zp : zero;
                xp += o + 1 < OWN ? a.x_st : (U - OWN + 1) * a.x_st;
                dtp += o + 1 < OWN ? a.dt_st : (U - OWN + 1) * a.dt_st;
                zp += o + 1 < OWN ? z_st : (U - OWN + 1) * z_st;
            }
        }
    };
    // The tile from row t0 on, into one of two places.
    const auto fetch_tile = [&](int t0, int place) {
        if constexpr (AHEAD) {
            constexpr int WIDE = 16 / sizeof(T), SIDE = CH / WIDE;  // channels of an access, accesses of a row
            const int first = g * per + ch0;
            const T* tensors[3] = {(const T*)a.x, (const T*)a.dt, gated ? (const T*)a.z : (const T*)a.x};
            const int64_t strides[3] = {a.x_st, a.dt_st, z_st};
#pragma unroll
            for (int input = 0; input < INPUTS; ++input)
#pragma unroll
                for (int i = 0; i < ROWS * SIDE; i += SCAN_THREADS) {
                    const int row = (i + tid) / SIDE, c = (i + tid) % SIDE * WIDE, t = t0 + row;
                    const bool in = t < end && ch0 + c < per;  // (per is a multiple of WIDE)
                    if (ROWS * SIDE % SCAN_THREADS == 0 || row < ROWS)
                        copy16(&s_in[place][input][row][c], tensors[input] + (in ? t * strides[input] + first + c : 0), in);
                }
            cp_async_commit();
        }
    };
    // And its elements of the next tile of B and C.
    T bcr[F];
    const auto fetch_bc = [&](int t0) {
#pragma unroll
        for (int f = 0; f < F; ++f) {
            const int i = f * SCAN_THREADS + tid, t = t0 + i / (2 * NP), n = i % NP;
            const bool is_c = i / NP % 2;
            const bool in = i < BC && t < end && (!PADDED || n < a.N) && !(CARRY && is_c);
            bcr[f] = in ? (is_c ? cp + t * a.c_st : bp + t * a.b_st)[n] : zero;
        }
    };
    const auto stage_bc = [&](int buffer) {
#pragma unroll
        for (int f = 0; f < F; ++f)
            if (f * SCAN_THREADS + tid < BC) (&s_bc[buffer][0][0][0])[f * SCAN_THREADS + tid] = to_f32(bcr[f]);
    };

    float total = 0.0f;
    int buffer = 0;
    // Rows t .. t + 3, in rows r0 .. of the tile; WHOLE: they and the four behind them are there.
    const auto group = [&](int t, int r0, auto whole) {
        float mine[OWN], mine_put[OWN], gate[OWN], skipped[OWN], step[U], put[U];
        if constexpr (AHEAD) {
#pragma unroll
            for (int o = 0; o < OWN; ++o) {
                xr[o] = s_in[buffer][0][r0 + own + o][tid / K];
                dtr[o] = s_in[buffer][1][r0 + own + o][tid / K];
                if (!CARRY) zr[o] = s_in[buffer][INPUTS - 1][r0 + own + o][tid / K];
            }
        }
#pragma unroll
        for (int o = 0; o < OWN; ++o) {
            const float x = to_f32(xr[o]);
            // rows behind the last one step by nothing: the states stay
            mine[o] = decltype(whole)::value || t + own + o < end ? step_width(to_f32(dtr[o]) + bias) : 0.0f;
            mine_put[o] = mine[o] * x;
            skipped[o] = skip * x;
            const float silu = fast_silu(to_f32(zr[o]));
            gate[o] = gated ? silu : 1.0f;
        }
        fetch(t + U, whole);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            step[u] = K == 1 ? mine[u % OWN] : __shfl_sync(0xffffffffu, mine[u % OWN], u / OWN * Sh::SHARE, K);
            put[u] = K == 1 ? mine_put[u % OWN] : __shfl_sync(0xffffffffu, mine_put[u % OWN], u / OWN * Sh::SHARE, K);
        }
        float y[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float4* b = reinterpret_cast<const float4*>(s_bc[buffer][r0 + u][0]) + lane;
            const float4* c = reinterpret_cast<const float4*>(s_bc[buffer][r0 + u][1]) + lane;
            const float2 st = make_float2(step[u], step[u]), pt = make_float2(put[u], put[u]);
            float2 acc = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int q = 0; q < SPT / 4; ++q) {
                if (PADDED && q >= fours) continue;
                const float4 b4 = b[q * K];
                const float4 c4 = CARRY ? b4 : c[q * K];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int j = 2 * q + i;
                    const float2 e = __fmul2_rn(st, rate[j]);
                    const float2 decay = make_float2(fast_exp2(e.x), fast_exp2(e.y));
                    float2 in = __fmul2_rn(pt, i ? make_float2(b4.z, b4.w) : make_float2(b4.x, b4.y));
                    if (PADDED == PAD_STATES && q == edge) {  // states that are not there stay 0, also when x is infinite
                        if (2 * i >= a.N % 4) in.x = 0.0f;
                        if (2 * i + 1 >= a.N % 4) in.y = 0.0f;
                    }
                    h[j] = __ffma2_rn(decay, h[j], in);
                    if (CARRY) continue;
                    const float2 ci = i ? make_float2(c4.z, c4.w) : make_float2(c4.x, c4.y);
                    acc = __ffma2_rn(h[j], ci, acc);
                }
            }
            y[u] = acc.x + acc.y;
            total += step[u];
        }
        if constexpr (!CARRY) {
            sum_rows<U, K>(y, lane);
#pragma unroll
            for (int o = 0; o < OWN; ++o) {
                if (open && lane % Sh::SHARE == 0 && (decltype(whole)::value || t + own + o < end))
                    *outp = from_f32<T>((y[o] + skipped[o]) * gate[o]);
                outp += o + 1 < OWN ? a.o_st : (U - OWN + 1) * a.o_st;
            }
        }
    };

    if (begin < end) {
        fetch_tile(begin, 0);
        fetch(begin, std::false_type());
        fetch_bc(begin);
        stage_bc(0);
    }
    for (int t0 = begin; t0 < end; t0 += ROWS, buffer ^= 1) {
        if (AHEAD) cp_async_wait<0>();
        __syncthreads();  // this tile is there, and the places of the one before are free
        const bool more = t0 + ROWS < end;
        if (more) {
            fetch_tile(t0 + ROWS, buffer ^ 1);
            fetch_bc(t0 + ROWS);
        }
        const int rows = min(ROWS, end - t0);
        for (int r0 = 0; r0 < rows; r0 += U) {
            if (end - (t0 + r0) >= 2 * U)
                group(t0 + r0, r0, std::true_type());
            else
                group(t0 + r0, r0, std::false_type());
        }
        if (more) stage_bc(buffer ^ 1);
    }

    float* kept = CARRY ? split.start + (int64_t)(piece.first + piece.at + 1) * a.D * a.N
                  : last && to >= 0 ? (float*)a.slot.state + to * a.slot.stride : nullptr;
    if (!open || !kept) return;
#pragma unroll
    for (int j = 0; j < SPT; ++j) {
        const int n = state_of(j);
        if (!PADDED || n < a.N) kept[(int64_t)d * a.N + n] = j % 2 ? h[j / 2].y : h[j / 2].x;
    }
    if (CARRY && lane == 0) split.sum[(int64_t)(piece.first + piece.at) * a.D + d] = total;
}

// Carries a split request's states from piece to piece: start[c] becomes the
// state that piece c starts from.  A thread a state, `blocks` blocks a request.
__global__ void __launch_bounds__(SCAN_THREADS) scan_carry_kernel(ScanArgs a, ScanSplit split, int blocks) {
    const int place = blockIdx.x / blocks;
    const int64_t at = (int64_t)(blockIdx.x - place * blocks) * SCAN_THREADS + threadIdx.x, size = (int64_t)a.D * a.N;
    const ScanPiece piece = find_piece<true>(a.cu, a.S, a.T, split.rows, place);
    if (piece.request < 0) return;
    const Span span = request_rows(a.cu, piece.request, a.T);
    int to, from;
    if (at >= size || !request_slots(a.slot, piece.request, to, from)) return;
    const int pieces = scan_pieces(span.end - span.begin, split.rows), d = (int)(at / a.N);
    if (piece.first < 0 || piece.first > split.room - pieces) return;
    const float rate = scan_rate(a.a[at]);
    float h = from >= 0 ? ((const float*)a.slot.state)[from * a.slot.stride + at] : 0.0f;
    float* start = split.start + piece.first * size + at;
    const float* sum = split.sum + (int64_t)piece.first * a.D + d;
    // (the loads of several pieces on their way together: one by one, each is waited for)
    start[0] = h;
    for (int c = 1; c < pieces; c += CARRY_AHEAD) {
        float own[CARRY_AHEAD], steps[CARRY_AHEAD];
#pragma unroll
        for (int i = 0; i < CARRY_AHEAD; ++i) {
            const int64_t at = min(c + i, pieces - 1);
            own[i] = start[at * size];
            steps[i] = sum[(at - 1) * a.D];
        }
#pragma unroll
        for (int i = 0; i < CARRY_AHEAD; ++i)
            if (c + i < pieces) {
                // (a decay that no float holds leaves an infinite state infinite, as its steps one by one do)
                h = fmaf(fmaxf(fast_exp2(rate * steps[i]), 1.17549435e-38f), h, own[i]);
                start[(int64_t)(c + i) * size] = h;
            }
    }
}

// ---------------------------------------------------------------- the launches
template <typename T, int K, int SPT, ScanPadding PADDED, bool SPLIT, bool AHEAD>
cudaError_t launch_scan(const ScanArgs& a, float* work, int piece_rows, cudaStream_t s) {
    using Sh = ScanShape<T, K, SPT, AHEAD>;
    const int64_t side = (int64_t)((a.D / a.G + Sh::CH - 1) / Sh::CH) * a.G;
    ScanSplit split{0, nullptr, nullptr, 0};
    int64_t pieces = a.S;
    if constexpr (SPLIT) {
        const int64_t room = scan_split_room(a.T, piece_rows), states = (int64_t)a.D * a.N;
        split = {piece_rows, work, work + room * states, (int)room};
        pieces = a.S + room;
        const int64_t blocks = (states + SCAN_THREADS - 1) / SCAN_THREADS;
        // that can be split and have room, whatever the offsets: each has more than SCAN_ALONE pieces
        const int64_t requests = room / (SCAN_ALONE + 1);
        if (side * room > INT32_MAX || blocks * requests > INT32_MAX) return cudaErrorInvalidValue;
        scan_kernel<T, K, SPT, PADDED, true, AHEAD><<<(unsigned)(side * room), SCAN_THREADS, 0, s>>>(a, split, (int)side);
        cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
        scan_carry_kernel<<<(unsigned)(blocks * requests), SCAN_THREADS, 0, s>>>(a, split, (int)blocks);
        e = cudaGetLastError();
        if (e != cudaSuccess) return e;
        add_launches(2);
    }
    if (side * pieces > INT32_MAX) return cudaErrorInvalidValue;
    scan_kernel<T, K, SPT, PADDED, false, AHEAD><<<(unsigned)(side * pieces), SCAN_THREADS, 0, s>>>(a, split, (int)side);
    add_launches(1);
    return cudaGetLastError();
}

template <typename T, int K, int SPT, bool SPLIT>
cudaError_t scan_padded(const ScanArgs& a, float* work, int rows, cudaStream_t s) {
    if (a.N % 4) return launch_scan<T, K, SPT, PAD_STATES, SPLIT, false>(a, work, rows, s);
    if (a.N != K * SPT) return launch_scan<T, K, SPT, PAD_FOURS, SPLIT, false>(a, work, rows, s);
    if constexpr (SPT == SCAN_LANE || K == 1) {
        const bool many = a.T > 1;
        if (a.D / a.G % (16 / sizeof(T)) == 0 && fits(a.x, many ? a.x_st : 0, 16, sizeof(T)) &&
            fits(a.dt, many ? a.dt_st : 0, 16, sizeof(T)) && fits(a.z, many && a.z ? a.z_st : 0, 16, sizeof(T)))
            return launch_scan<T, K, SPT, PAD_NONE, SPLIT, true>(a, work, rows, s);
    }
    return launch_scan<T, K, SPT, PAD_NONE, SPLIT, false>(a, work, rows, s);
}

// Lanes of SCAN_LANE states; of four when the blocks of those would leave
// multiprocessors without one.
template <typename T>
cudaError_t scan_type(const ScanArgs& a, float* work, const ScanPlan& plan, cudaStream_t s) {
    if (plan.rows > 0) {
        if (a.N <= 4) return scan_padded<T, 1, 4, true>(a, work, plan.rows, s);
        if (a.N <= 8) return scan_padded<T, 1, 8, true>(a, work, plan.rows, s);
        if (a.N <= 16) return scan_padded<T, 1, SCAN_LANE, true>(a, work, plan.rows, s);
        if (a.N <= 32) return scan_padded<T, 2, SCAN_LANE, true>(a, work, plan.rows, s);
        if (a.N <= 64) return scan_padded<T, 4, SCAN_LANE, true>(a, work, plan.rows, s);
        if (a.N <= 128) return scan_padded<T, 8, SCAN_LANE, true>(a, work, plan.rows, s);
        return scan_padded<T, 16, SCAN_LANE, true>(a, work, plan.rows, s);
    }
    if (a.N <= 4) return scan_padded<T, 1, 4, false>(a, work, 0, s);
    if (plan.thin) {
        if (a.N <= 8) return scan_padded<T, 2, 4, false>(a, work, 0, s);
        if (a.N <= 16) return scan_padded<T, 4, 4, false>(a, work, 0, s);
        if (a.N <= 32) return scan_padded<T, 8, 4, false>(a, work, 0, s);
        if (a.N <= 64) return scan_padded<T, 16, 4, false>(a, work, 0, s);
        if (a.N <= 128) return scan_padded<T, 32, 4, false>(a, work, 0, s);
    }
    if (a.N <= 8) return scan_padded<T, 1, 8, false>(a, work, 0, s);
    if (a.N <= 16) return scan_padded<T, 1, SCAN_LANE, false>(a, work, 0, s);
    if (a.N <= 32) return scan_padded<T, 2, SCAN_LANE, false>(a, work, 0, s);
    if (a.N <= 64) return scan_padded<T, 4, SCAN_LANE, false>(a, work, 0, s);
    if (a.N <= 128) return scan_padded<T, 8, SCAN_LANE, false>(a, work, 0, s);
    return scan_padded<T, 16, SCAN_LANE, false>(a, work, 0, s);
}

}  // namespace
}  // namespace krk
