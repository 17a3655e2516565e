/**
 * Rotary positions: pair (a, b) of a head's elements becomes (a cos - b sin, b cos + a sin) with the angle position * frequency;
 * the gradient is the same with -sin. Every head of a token turns alike.
 *
 * Two reads or writes of memory per element and a handful of operations: HBM bounds it. Angles are computed here and not read from
 * a table, so that no position lies outside of one: in 64 bits, since 32 hold no fraction of a turn at position 10^6, as
 * turns whose whole part is dropped before the sine and cosine in 32. A CTA takes a few tokens, computes their angles
 * once into shared memory and then walks over their heads.
 */
#include "decoder_ops.hpp"
#include "launch_early.cuh"
#include "row_access.cuh"

namespace dccl {

struct RotaryArgs {
    DcclHeads q, k;
    const double* freqs;
    const void* positions;
    long long pos_batch, pos_seq, first;
    size_t tokens;
    unsigned seq, head_dim, pairs, per_cta;
    bool interleaved, back, wide_positions;
    float scale;
};

constexpr int kRotaryThreads = 256;
constexpr unsigned kRotaryPairs = 1024;     // pairs of the tokens of one CTA: 8 KB of shared memory

/** P: elements per access. An item is two accesses: both halves of P pairs, or 2 P elements of what is only copied. */
template <typename T, int P>
__global__ void __launch_bounds__(kRotaryThreads) k_rotary(const __grid_constant__ RotaryArgs a) {
    wait_for_stream();
    __shared__ float cosines[kRotaryPairs], sines[kRotaryPairs];
    const size_t first = (size_t)blockIdx.x * a.per_cta;
    const unsigned n = (unsigned)(a.tokens - first < a.per_cta ? a.tokens - first : a.per_cta);
    for (unsigned i = threadIdx.x; i < n * a.pairs; i += kRotaryThreads) {
        const size_t token = first + i / a.pairs;
        const long long b = (long long)(token / a.seq), s = (long long)(token % a.seq);
        long long pos = a.first + s;
        if (a.positions) {
            const long long at = b * a.pos_batch + s * a.pos_seq;
            pos = a.wide_positions ? reinterpret_cast<const long long*>(a.positions)[at] : reinterpret_cast<const int*>(a.positions)[at];
        }
        const double turns = (double)pos * (a.freqs[i % a.pairs] * 0.15915494309189533577);      // 1 / (2 pi)
        float sn, cs;
        sincospif(2.0f * (float)(turns - rint(turns)), &sn, &cs);
        cosines[i] = cs * a.scale;
        sines[i] = (a.back ? -sn : sn) * a.scale;
    }
    __syncthreads();
    const unsigned turned = a.pairs / P, copied = (a.head_dim - 2 * a.pairs) / P, per_head = turned + (copied + 1) / 2;
    const unsigned heads = a.q.heads + a.k.heads, per_token = heads * per_head;
    for (unsigned i = threadIdx.x; i < n * per_token; i += kRotaryThreads) {
        const unsigned local = i / per_token, h = i % per_token / per_head, j = i % per_head;
        const size_t token = first + local;
        const long long b = (long long)(token / a.seq), s = (long long)(token % a.seq);
        const bool in_q = h < (unsigned)a.q.heads;
        const DcclHeads& x = in_q ? a.q : a.k;
        const long long hh = in_q ? h : h - a.q.heads;
        const T* from = reinterpret_cast<const T*>(x.in) + b * x.in_batch + s * x.in_seq + hh * x.in_head;
        T* to = reinterpret_cast<T*>(x.out) + b * x.out_batch + s * x.out_seq + hh * x.out_head;
        if (j < turned) {
            const unsigned lo = a.interleaved ? 2 * j * P : j * P, hi = a.interleaved ? lo + P : a.pairs + lo;
            const Run<T, P> u = ld_run<T, P>(from + lo), v = ld_run<T, P>(from + hi);
            const float *cs = cosines + local * a.pairs + j * P, *sn = sines + local * a.pairs + j * P;
            float e[2 * P];
#pragma unroll
            for (int p = 0; p < P; p++) { e[p] = Traits<T>::up(u.e[p]); e[P + p] = Traits<T>::up(v.e[p]); }
            Run<T, P> ou, ov;
#pragma unroll
            for (int p = 0; p < P; p++) {
                const float c = cs[p], d = sn[p];
                if (a.interleaved) {
                    const T even = Traits<T>::down(e[2 * p] * c - e[2 * p + 1] * d), odd = Traits<T>::down(e[2 * p + 1] * c + e[2 * p] * d);
                    if (P == 1) { ou.e[0] = even; ov.e[0] = odd; }
                    else if (p < P / 2) { ou.e[2 * p % P] = even; ou.e[(2 * p + 1) % P] = odd; }
                    else { ov.e[2 * p % P] = even; ov.e[(2 * p + 1) % P] = odd; }
                } else {
                    ou.e[p] = Traits<T>::down(e[p] * c - e[P + p] * d);
                    ov.e[p] = Traits<T>::down(e[P + p] * c + e[p] * d);
                }
            }
            st_run<T, P>(to + lo, ou);
            st_run<T, P>(to + hi, ov);
        } else {
            const unsigned at = 2 * a.pairs + (j - turned) * 2 * P;
            const bool two = at + P < a.head_dim;
            const Run<T, P> u = ld_run<T, P>(from + at);
            Run<T, P> v;
            if (two) v = ld_run<T, P>(from + at + P);
            st_run<T, P>(to + at, u);
            if (two) st_run<T, P>(to + at + P, v);
        }
    }
}

/** Whether every access of P elements of `size` bytes falls on its own size. */
static bool rotary_runs(const DcclHeads& x, int p, int size) {
    if (!x.heads) return true;
    if (!aligned_to((size_t)p * size, {x.in, x.out})) return false;
    return (x.in_batch | x.in_seq | x.in_head | x.out_batch | x.out_seq | x.out_head) % p == 0;
}

template <typename T> static cudaError_t rotary_launch(int p, unsigned grid, cudaStream_t stream, const RotaryArgs& a) {
    switch (p) {
        case 8: if constexpr (sizeof(T) == 2) return launch_early(k_rotary<T, 8>, grid, kRotaryThreads, stream, a); else return cudaErrorInvalidValue;
        case 4: return launch_early(k_rotary<T, 4>, grid, kRotaryThreads, stream, a);
        case 2: return launch_early(k_rotary<T, 2>, grid, kRotaryThreads, stream, a);
        default: return launch_early(k_rotary<T, 1>, grid, kRotaryThreads, stream, a);
    }
}

} // namespace dccl

using namespace dccl;

extern "C" int dccl_rotary(int device, int dtype, size_t batch, size_t seq, int head_dim, int pairs, int interleaved, int back, const DcclHeads* q, const DcclHeads* k,
                           const double* freqs, const void* positions, int positions64, long long pos_batch, long long pos_seq, long long first, double scale,
                           void* stream_v) {
    const size_t tokens = batch * seq;
    if (!tokens || !head_dim || q->heads + k->heads == 0) return 0;
    if (pairs < 1 || 2 * pairs > head_dim || (unsigned)pairs > kRotaryPairs || seq > 0xffffffffu || q->heads < 0 || k->heads < 0
        || (long long)(q->heads + k->heads) * head_dim > (1 << 24))
        return report("dccl_rotary", cudaErrorInvalidValue);
    const int size = dtype == 7 ? 4 : 2;
    int p = 16 / size;
    while (p > 1 && (pairs % p || (head_dim - 2 * pairs) % p || !rotary_runs(*q, p, size) || !rotary_runs(*k, p, size))) p /= 2;
    // tokens of a CTA: two items per thread, as long as that leaves enough CTAs
    const size_t items = (size_t)(q->heads + k->heads) * ((pairs / p) + ((head_dim - 2 * pairs) / p + 1) / 2);
    size_t per = 2 * kRotaryThreads / (items ? items : 1);
    const size_t sms = (size_t)sm_count(device);
    if (per > tokens / (sms ? 4 * sms : 1)) per = tokens / (sms ? 4 * sms : 1);
    if (per > kRotaryPairs / pairs) per = kRotaryPairs / pairs;
    if (!per) per = 1;
    const size_t grid = (tokens + per - 1) / per;
    if (grid > 0x7fffffffu) return report("dccl_rotary", cudaErrorInvalidValue);
    const RotaryArgs a = {*q, *k, freqs, positions, pos_batch, pos_seq, first, tokens, (unsigned)seq, (unsigned)head_dim, (unsigned)pairs, (unsigned)per,
                          interleaved != 0, back != 0, positions64 != 0, (float)scale};
    cudaStream_t stream = (cudaStream_t)stream_v;
    OnDevice on(device);
    if (on.e != cudaSuccess) return report("dccl_rotary", on.e);
    return report("dccl_rotary", dtype == 6 ? rotary_launch<__half>(p, (unsigned)grid, stream, a) : dtype == 7 ? rotary_launch<float>(p, (unsigned)grid, stream, a)
                                 : dtype == 9 ? rotary_launch<__nv_bfloat16>(p, (unsigned)grid, stream, a) : cudaErrorInvalidValue);
}
