/**
 * Rotary positions: pair (a, b) of a head's elements becomes (a cos - b sin, b cos + a sin) with the angle position * frequency;
 * the gradient is the same with -sin. Every head of a token turns alike.
 *
 * Two reads or writes of memory per element and a handful of operations: HBM bounds it. Angles are computed here and not read from
 * a table, so that no position lies outside of one: in 64 bits, since 32 hold no fraction of a turn at position 10^6, as
 * turns whose whole part is dropped before the sine and cosine in 32, to which what the rounding of the rest took off is added. A CTA takes consecutive tokens of one sequence and computes their
 * angles, each once, into shared memory. A thread keeps its place within a token, its head and its elements, and walks along the
 * tokens with the loads of two or four of them in flight, the first under way while the angles are computed: what it takes to find an
 * element, as many instructions as to turn it, is paid once for all tokens.
 *
 * 16384 tokens x 36 heads x 64 bf16: 32 us each way (4.7 TB/s), 46 with a thread for each place of each token; 5003 x 24 x 80 fp32, 17 pairs of
 * neighbours: 17 us (4.5 TB/s).
 */
#include "decoder_ops.hpp"
#include "../kernels/launch_early.cuh"
#include "row_access.cuh"

namespace dccl {

struct RotaryArgs {
    DcclHeads q, k;
    const double* freqs;
    const void* positions;
    long long pos_batch, pos_seq, first;
    unsigned seq, head_dim, pairs;
    unsigned chunk, at_once;            // tokens of a CTA, and those that its threads cover at a time
    Divisor chunks;                     // of a sequence
    Divisor table;                      // pairs of a token in shared memory: a multiple of four, the last ones without a value
    Divisor items, per_head;            // places of a token and of a head
    bool back, wide_positions;
    float scale;
};

constexpr unsigned kRotaryThreads = 512;            // at most
constexpr unsigned kRotaryPairs = 2048;             // of the tokens of a CTA: 16 KB of shared memory

template <int N> __device__ __forceinline__ void ld_floats(float (&f)[N], const float* p) {
#pragma unroll
    for (int i = 0; i < N; i++) f[i] = p[i];
}
template <> __device__ __forceinline__ void ld_floats<4>(float (&f)[4], const float* p) {
    const Run<float, 4> r = ld_run<float, 4>(p);
#pragma unroll
    for (int i = 0; i < 4; i++) f[i] = r.e[i];
}
template <> __device__ __forceinline__ void ld_floats<8>(float (&f)[8], const float* p) {
    const Run<float, 4> r = ld_run<float, 4>(p), q = ld_run<float, 4>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; i++) { f[i] = r.e[i]; f[4 + i] = q.e[i]; }
}

/**
 * P: elements per access. INTERLEAVED: a place in a head is one access, or for P = 1 two, of whole pairs. Otherwise it is two: the
 * first and the second elements of P pairs, or 2 P elements that are only copied.
 */
template <typename T, int P, bool INTERLEAVED>
__global__ void __launch_bounds__(kRotaryThreads, 2) k_rotary(const __grid_constant__ RotaryArgs a) {
    wait_for_stream();
    constexpr bool kTwo = !INTERLEAVED || P == 1;
    constexpr int kPairs = INTERLEAVED && P > 1 ? P / 2 : P;                            // of a place
    extern __shared__ float4 angles[];                                                  // cosines of each token's pairs, then sines
    const unsigned batch = a.chunks.quotient(blockIdx.x), begin = (blockIdx.x - batch * a.chunks.d) * a.chunk;
    const unsigned n = a.seq - begin < a.chunk ? a.seq - begin : a.chunk;
    const unsigned sub = a.at_once > 1 ? a.items.quotient(threadIdx.x) : 0;
    const unsigned turned = (a.pairs + kPairs - 1) / kPairs;                            // places of a head that turn, wholly or in part
    constexpr int kAhead = kTwo && P * sizeof(T) == 16 ? 2 : 4;                         // tokens of a thread in flight
    struct Access { Run<T, P> u, v; } x[kAhead];
    unsigned j, gap;
    bool two;
    const T* from;
    T* to;
    long long in_step, out_step;
    const auto take = [&](unsigned item) {
        const unsigned h = a.per_head.quotient(item);
        j = item - h * a.per_head.d;
        const bool in_q = h < (unsigned)a.q.heads;
        const DcclHeads& x = in_q ? a.q : a.k;
        const unsigned head = in_q ? h : h - a.q.heads;
        const unsigned lo = INTERLEAVED ? j * (P == 1 ? 2 : P) : j < turned ? j * P : 2 * a.pairs + (j - turned) * 2 * P;
        gap = !INTERLEAVED && j < turned ? a.pairs : P;
        two = kTwo && lo + gap < a.head_dim;
        from = reinterpret_cast<const T*>(x.in) + batch * x.in_batch + (begin + sub) * x.in_seq + head * x.in_head + lo;
        to = reinterpret_cast<T*>(x.out) + batch * x.out_batch + (begin + sub) * x.out_seq + head * x.out_head + lo;
        in_step = a.at_once * x.in_seq;
        out_step = a.at_once * x.out_seq;
    };
    const auto load = [&](Access& x, unsigned t) {
        if (t < n) {
            x.u = ld_run<T, P>(from);
            if (kTwo && two) x.v = ld_run<T, P>(from + gap);
        }
        from += in_step;
    };
    const unsigned step = a.at_once;
    const auto load_first = [&](unsigned item) {
        take(item);
#pragma unroll
        for (int r = 0; r < kAhead; r++) load(x[r], sub + r * step);
    };
    float* const cosines = reinterpret_cast<float*>(angles);
    float* const sines = cosines + n * a.table.d;
    const auto turn = [&](Access& x, unsigned t) {
        if (t >= n) return;
        if (j < turned) {
            float c[kPairs], s[kPairs], x0[P], x1[P];
            ld_floats<kPairs>(c, cosines + t * a.table.d + j * kPairs);
            ld_floats<kPairs>(s, sines + t * a.table.d + j * kPairs);
            if constexpr (INTERLEAVED && P > 1) {
#pragma unroll
                for (int e = 0; e < P / 2; e++) {
                    const float even = Traits<T>::up(x.u.e[2 * e]), odd = Traits<T>::up(x.u.e[2 * e + 1]);
                    x0[2 * e] = even * c[e] - odd * s[e];
                    x0[2 * e + 1] = odd * c[e] + even * s[e];
                }
                const Run<T, P> whole = round_run<T, P>(x0);
#pragma unroll
                for (int e = 0; e < P; e++)
                    if (j * kPairs + e / 2 < a.pairs) x.u.e[e] = whole.e[e];
            } else {
#pragma unroll
                for (int e = 0; e < P; e++) {
                    const float p = Traits<T>::up(x.u.e[e]), q = Traits<T>::up(x.v.e[e]);
                    x0[e] = p * c[e] - q * s[e];
                    x1[e] = q * c[e] + p * s[e];
                }
                x.u = round_run<T, P>(x0);
                x.v = round_run<T, P>(x1);
            }
        }
        st_run<T, P>(to, x.u);
        if (kTwo && two) st_run<T, P>(to + gap, x.v);
        to += out_step;
    };
    unsigned item = sub < a.at_once ? threadIdx.x - sub * a.items.d : a.items.d;
    if (item < a.items.d) load_first(item);
    for (unsigned k = threadIdx.x; k < n * a.table.d; k += blockDim.x) {
        const unsigned of = a.table.quotient(k), pair = k - of * a.table.d;
        if (pair >= a.pairs) continue;
        long long pos = a.first + begin + of;
        if (a.positions) {
            const long long at = batch * a.pos_batch + (begin + of) * a.pos_seq;
            pos = a.wide_positions ? reinterpret_cast<const long long*>(a.positions)[at] : reinterpret_cast<const int*>(a.positions)[at];
        }
        const double turns = (double)pos * (a.freqs[pair] * 0.15915494309189533577), part = turns - rint(turns);      // 1 / (2 pi)
        const float near = (float)part, rest = (float)(part - near) * 6.2831853f;      // what rounding took off, in radians: under 2^-23, so its square is nothing
        float s0, c0;
        sincospif(2.0f * near, &s0, &c0);
        const float sn = fmaf(c0, rest, s0), cs = fmaf(-s0, rest, c0);
        cosines[k] = cs * a.scale;
        sines[k] = (a.back ? -sn : sn) * a.scale;
    }
    __syncthreads();
    while (item < a.items.d) {
        for (unsigned t = sub; t < n; t += kAhead * step)
#pragma unroll
            for (int r = 0; r < kAhead; r++) {
                turn(x[r], t + r * step);
                load(x[r], t + (r + kAhead) * step);
            }
        item += a.at_once > 1 ? a.items.d : blockDim.x;
        if (item < a.items.d) load_first(item);
    }
}

/** Whether every access of P elements of `size` bytes falls on its own size. */
static bool rotary_runs(const DcclHeads& x, int p, int size) {
    if (!x.heads) return true;
    if (!aligned_to((size_t)p * size, {x.in, x.out})) return false;
    return (x.in_batch | x.in_seq | x.in_head | x.out_batch | x.out_seq | x.out_head) % p == 0;
}

template <typename T, bool INTERLEAVED> static cudaError_t rotary_launch(int p, unsigned grid, unsigned block, size_t shared, cudaStream_t stream, const RotaryArgs& a) {
    switch (p) {
        case 8: if constexpr (sizeof(T) == 2) return launch_early_shared(k_rotary<T, 8, INTERLEAVED>, grid, block, shared, stream, a); else return cudaErrorInvalidValue;
        case 4: return launch_early_shared(k_rotary<T, 4, INTERLEAVED>, grid, block, shared, stream, a);
        case 2: return launch_early_shared(k_rotary<T, 2, INTERLEAVED>, grid, block, shared, stream, a);
        default: return launch_early_shared(k_rotary<T, 1, INTERLEAVED>, grid, block, shared, stream, a);
    }
}
template <typename T> static cudaError_t rotary_launch(bool interleaved, int p, unsigned grid, unsigned block, size_t shared, cudaStream_t stream, const RotaryArgs& a) {
    return interleaved ? rotary_launch<T, true>(p, grid, block, shared, stream, a) : rotary_launch<T, false>(p, grid, block, shared, stream, a);
}

} // namespace dccl

using namespace dccl;

extern "C" int dccl_rotary(int device, int dtype, size_t batch, size_t seq, int head_dim, int pairs, int interleaved, int back, const DcclHeads* q, const DcclHeads* k,
                           const double* freqs, const void* positions, int positions64, long long pos_batch, long long pos_seq, long long first, double scale,
                           void* stream_v) {
    if (!batch || !seq || !head_dim || q->heads + k->heads == 0) return 0;
    const size_t limit = (1u << 31) - 1, tokens = batch * seq;
    if (pairs < 1 || 2 * pairs > head_dim || pairs > DCCL_ROTARY_MAX_PAIRS || batch > limit || seq > limit || tokens > limit || q->heads < 0 || k->heads < 0
        || (long long)(q->heads + k->heads) * head_dim > DCCL_ROTARY_MAX_TOKEN)
        return report("dccl_rotary", cudaErrorInvalidValue);
    const int size = dtype == 7 ? 4 : 2, rest = head_dim - 2 * pairs;
    int p = 16 / size;
    // pairs of neighbours lie within an access, and what does not turn may share one with them
    while (p > 1 && ((interleaved ? head_dim % p : pairs % p || rest % p) || !rotary_runs(*q, p, size) || !rotary_runs(*k, p, size))) p /= 2;
    const unsigned heads = (unsigned)(q->heads + k->heads);
    const unsigned per_head = interleaved ? (p == 1 ? (unsigned)(head_dim + 1) / 2 : (unsigned)(head_dim / p)) : (unsigned)(pairs / p + (rest / p + 1) / 2);
    const unsigned items = heads * per_head, table = (unsigned)(pairs + 3) / 4 * 4;
    // several small tokens at once, or one large one in a few rounds, by about 256 threads
    unsigned at_once = items < 192 ? (256 + items / 2) / items : 1;
    const unsigned rounds = (items + kRotaryThreads - 1) / kRotaryThreads;
    if (at_once > seq) at_once = (unsigned)seq;
    const unsigned block = at_once > 1 ? (at_once * items + 31) / 32 * 32 : ((items + rounds - 1) / rounds + 31) / 32 * 32;
    // one wave of CTAs, where their angles fit into shared memory
    const size_t resident = (size_t)sm_count(device) * (1024 / block), want = resident / batch ? resident / batch : 1;
    size_t chunk = (seq + want - 1) / want;
    if (chunk < at_once) chunk = at_once;
    if (chunk > kRotaryPairs / table) chunk = kRotaryPairs / table;
    const size_t chunks = (seq + chunk - 1) / chunk, grid = batch * chunks;
    if (grid > limit) return report("dccl_rotary", cudaErrorInvalidValue);
    const RotaryArgs a = {*q, *k, freqs, positions, pos_batch, pos_seq, first, (unsigned)seq, (unsigned)head_dim, (unsigned)pairs, (unsigned)chunk, at_once, Divisor((unsigned)chunks),
                          Divisor(table), Divisor(items), Divisor(per_head), back != 0, positions64 != 0, (float)scale};
    const size_t shared = chunk * table * 2 * sizeof(float);
    const bool i = interleaved != 0;
    cudaStream_t stream = (cudaStream_t)stream_v;
    OnDevice on(device);
    if (on.e != cudaSuccess) return report("dccl_rotary", on.e);
    return report("dccl_rotary", dtype == 6 ? rotary_launch<__half>(i, p, (unsigned)grid, block, shared, stream, a) : dtype == 7 ? rotary_launch<float>(i, p, (unsigned)grid, block, shared, stream, a)
                                 : dtype == 9 ? rotary_launch<__nv_bfloat16>(i, p, (unsigned)grid, block, shared, stream, a) : cudaErrorInvalidValue);
}
