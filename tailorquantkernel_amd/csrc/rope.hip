// rope.hip — rotary positions for long contexts: the cos and sin rows that every
// other call takes, at any positions and with the scalings that carry a model past
// its trained length (tq_hip_rope_rows), and a projection's q and k heads normalized
// and turned in one pass (tq_hip_norm_rope).  The reference has plain RoPE on a host
// table (model/rope.c:4-29), in fp32, and RMSNorm apart (model/rmsnorm.c:4-19).
//
//   pair i of R / 2:  f_i = theta^(-2 i / R), scaled;  cos, sin = m cos, m sin(pos f_i)
//   head:             y = x / sqrt(eps + mean x^2) * w;  (a, b) -> (a c - b s, a s + b c)
//
// An angle is up to 2^31 radians, of which fp32 would keep nothing, so it is made in
// 64 bits: pos f_i is off by half a step of fp64, k = rint(angle 2 / pi) leaves
// angle - k pi / 2 by two fused products with pi / 2 in two parts, and Taylor's series
// on [-pi/4, pi/4] (to r^11 and r^12: below 2^-33) are rounded to fp32 once.  fp64 runs
// at the rate of fp32 here and a row's angles are made once for all its heads.
#include <math.h>

#include <algorithm>

#include "tq_common.hpp"

namespace {

using namespace tq;

constexpr int kMaxPairs = 128;

struct Frequencies {
    double f[kMaxPairs];   // radians per position
    double magnitude;
    int pairs;
};

struct CosSin {
    float c, s;
};

__device__ __forceinline__ CosSin cos_sin(int pos, double f, double magnitude) {
    constexpr double kTwoByPi = 0.63661977236758134308;
    constexpr double kHalfPi = 1.57079632679489661923, kHalfPiLow = 6.12323399573676603587e-17;
    const double x = (double)pos * f;
    const double k = rint(x * kTwoByPi);
    const double r = fma(-k, kHalfPiLow, fma(-k, kHalfPi, x)), z = r * r;
    double s = -1.0 / 39916800.0;
    s = fma(s, z, 1.0 / 362880.0);
    s = fma(s, z, -1.0 / 5040.0);
    s = fma(s, z, 1.0 / 120.0);
    s = fma(s, z, -1.0 / 6.0);
    s = fma(s * z, r, r);
    double c = 1.0 / 479001600.0;
    c = fma(c, z, -1.0 / 3628800.0);
    c = fma(c, z, 1.0 / 40320.0);
    c = fma(c, z, -1.0 / 720.0);
    c = fma(c, z, 1.0 / 24.0);
    c = fma(c, z, -0.5);
    c = fma(c, z, 1.0);
    const int quadrant = (int)k & 3;
    const double cc = quadrant & 1 ? s : c, ss = quadrant & 1 ? c : s;
    return {(float)(magnitude * (((quadrant + 1) & 2) ? -cc : cc)), (float)(magnitude * ((quadrant & 2) ? -ss : ss))};
}

// Four consecutive values of the flat [n][pairs] arrays per thread.  Bound by the launch
// (64 rows of 64 pairs in 2.8 us) and by the angles and the stores alike (32,768 rows, 17 MB,
// in 7.3).
__global__ __launch_bounds__(256) void rope_rows_kernel(Frequencies a, const int32_t *pos, size_t total, float *cos_t,
                                                        float *sin_t) {
    const size_t at = 4 * ((size_t)blockIdx.x * 256 + threadIdx.x);
    if (at >= total) return;
    size_t row = at / (unsigned)a.pairs;
    int i = (int)(at - row * a.pairs);
    const int count = (int)min((size_t)4, total - at);
    float c[4], s[4];
    int p = pos ? pos[row] : (int)row;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        c[j] = s[j] = 0.0f;
        if (j < count) {
            const CosSin v = cos_sin(p, a.f[i], a.magnitude);
            c[j] = v.c;
            s[j] = v.s;
            if (++i == a.pairs && j + 1 < count) {
                i = 0;
                row++;
                p = pos ? pos[row] : (int)row;
            }
        }
    }
    if (count == 4) {
        *reinterpret_cast<v4f_any *>(cos_t + at) = v4f_any{c[0], c[1], c[2], c[3]};
        *reinterpret_cast<v4f_any *>(sin_t + at) = v4f_any{s[0], s[1], s[2], s[3]};
    } else {
        for (int j = 0; j < count; j++) {
            cos_t[at + j] = c[j];
            sin_t[at + j] = s[j];
        }
    }
}

struct NormRopeArgs {
    Frequencies freq;
    const int32_t *pos;
    tq_hip_heads q, k;       // k's heads follow q's
    int heads;               // of both
    int head_dim, rot;
    float eps;
};

// Sum over the LANES lanes of a head, the same value in each.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float x) {
    x += dpp_f<kDppQuadXor1>(x);
    x += dpp_f<kDppQuadXor2>(x);
    x += dpp_f<kDppRowHalfMirror>(x);
    if constexpr (LANES >= 16) x += dpp_f<kDppRowMirror>(x);
    if constexpr (LANES >= 32) {
        const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    }
    if constexpr (LANES >= 64) {
        const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
        x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    }
    return x;
}

// Grid (row, chunk of U * 256 / LANES heads): LANES lanes have a head, values 4 l .. 4 l + 3
// each.  The partners of neighbouring pairs are in the lane (rot a multiple of 4), those
// of halves in another lane of the wave (a multiple of 8); otherwise a lane reads its
// partners too, which is rare enough.  A head lies in one wave, whose loads all come before
// its stores: in place is safe either way.
//   Bound by reading and writing the heads: 4,096 rows of 64 and 8 heads of 128 (302 MB) in
// 67 us, 8,192 in 124 (4.9 TB/s, where a copy of as much reaches 5.3), 64 rows of 32 and 8
// in 6.5, the launch and the angles.  Rotary dims that are no such multiples take 111-115
// us for 4,096 rows, a lane's four partners one by one.  Stores past the caches
// (nontemporal) took 2,048 rows from 36 to 24 us and 4,096 from 72; loads past them undo
// that (34).
enum { kHalves, kNeighbours, kAny };
template <int LANES, int U, int FORM>
__global__ __launch_bounds__(256) void norm_rope_kernel(NormRopeArgs a, int interleaved) {
    __shared__ float cs[kMaxPairs], sn[kMaxPairs];
    constexpr int PER = 256 / LANES;
    const int tid = threadIdx.x, l = tid % LANES;
    const size_t row = blockIdx.x;
    const int hd = a.head_dim, rot = a.rot;
    const bool in = 4 * l < hd;
    const bool turns = 4 * l < rot, upper = 8 * l >= rot;
    // (FORM kHalves) the lane of this lane's partners
    const int other = (tid & 63) + (!turns ? 0 : upper ? -rot / 8 : rot / 8);
    // (FORM kAny) the partner of value 4 l + j
    int mate[4];
    if constexpr (FORM == kAny) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int e = 4 * l + j;
            mate[j] = e >= rot || !in ? min(e, hd - 1) : interleaved ? e ^ 1 : e < rot / 2 ? e + rot / 2 : e - rot / 2;
        }
    }
    float x[U][4], y[U][4];
    const float *weight[U];
    float *out[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int head = (blockIdx.y * U + u) * PER + tid / LANES;
        const bool of_q = head < a.q.heads;
        const tq_hip_heads &t = of_q ? a.q : a.k;
        const int h = of_q ? head : head - a.q.heads;
        weight[u] = t.norm;
        out[u] = head < a.heads && in ? t.out + row * t.out_stride + (size_t)h * hd : nullptr;
#pragma unroll
        for (int j = 0; j < 4; j++) x[u][j] = y[u][j] = 0.0f;
        if (out[u]) {
            const float *src = t.x + row * t.stride + (size_t)h * hd;
            const v4f_any v = *reinterpret_cast<const v4f_any *>(src + 4 * l);
            x[u][0] = v.x, x[u][1] = v.y, x[u][2] = v.z, x[u][3] = v.w;
            if constexpr (FORM == kAny) {
#pragma unroll
                for (int j = 0; j < 4; j++) y[u][j] = src[mate[j]];
            }
        }
    }
    // the row's angles, while the heads are on their way
    const int p = a.pos ? a.pos[row] : (int)row;
    if (tid < rot / 2) {
        const CosSin v = cos_sin(p, a.freq.f[tid], a.freq.magnitude);
        cs[tid] = v.c;
        sn[tid] = v.s;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; u++) {
        const float sum = lanes_sum<LANES>((x[u][0] * x[u][0] + x[u][1] * x[u][1]) + (x[u][2] * x[u][2] + x[u][3] * x[u][3]));
        if (weight[u] && out[u]) {
            const float inv = 1.0f / sqrtf(a.eps + sum / (float)hd);
            const float *w = weight[u];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                x[u][j] = x[u][j] * inv * w[4 * l + j];
                if constexpr (FORM == kAny) y[u][j] = y[u][j] * inv * w[mate[j]];
            }
        }
        float *v = x[u];
        if constexpr (FORM == kHalves) {
#pragma unroll
            for (int j = 0; j < 4; j++) y[u][j] = __shfl(v[j], other);
        }
        if (!out[u]) continue;
        if constexpr (FORM == kAny) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int e = 4 * l + j;
                if (e >= rot) continue;
                const int i = interleaved ? e / 2 : e % (rot / 2);
                const bool lower = interleaved ? !(e & 1) : e < rot / 2;
                v[j] = lower ? v[j] * cs[i] - y[u][j] * sn[i] : y[u][j] * sn[i] + v[j] * cs[i];
            }
        } else if (turns && FORM == kHalves) {
            const int i = 4 * l - (upper ? rot / 2 : 0);
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = v[j] * cs[i + j] + y[u][j] * (upper ? sn[i + j] : -sn[i + j]);
        } else if (turns) {
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
                const float c = cs[2 * l + j / 2], s = sn[2 * l + j / 2], p0 = v[j], p1 = v[j + 1];
                v[j] = p0 * c - p1 * s;
                v[j + 1] = p0 * s + p1 * c;
            }
        }
        const v4f_any r{v[0], v[1], v[2], v[3]};
        __builtin_nontemporal_store(r, reinterpret_cast<v4f_any *>(out[u] + 4 * l));
    }
}

// The frequencies of a descriptor, or false where it is not one.
bool frequencies(const tq_hip_rope *r, Frequencies &out) {
    const double pi = 3.14159265358979323846;
    if (!r || r->rotary_dim < 2 || r->rotary_dim % 2 || r->rotary_dim > 2 * kMaxPairs) return false;
    if (r->layout != TQ_HIP_ROPE_HALF && r->layout != TQ_HIP_ROPE_INTERLEAVED) return false;
    if (!(r->theta >= 1.0) || !isfinite(r->theta)) return false;
    const int kind = r->scaling, R = r->rotary_dim;
    if (kind < TQ_HIP_ROPE_PLAIN || kind > TQ_HIP_ROPE_YARN) return false;
    if (kind != TQ_HIP_ROPE_PLAIN && (!(r->factor >= 1.0) || !isfinite(r->factor))) return false;
    if (kind == TQ_HIP_ROPE_BANDS && !(r->trained_len > 0 && r->high > r->low && r->low >= 0.0 && isfinite(r->high)))
        return false;
    if (kind == TQ_HIP_ROPE_YARN &&
        !(r->trained_len > 0 && r->high >= r->low && r->low > 0.0 && isfinite(r->high) && r->theta > 1.0 &&
          r->magnitude >= 0.0 && isfinite(r->magnitude)))
        return false;
    const double s = r->factor, theta = kind == TQ_HIP_ROPE_NTK && R > 2 ? r->theta * pow(s, R / (R - 2.0)) : r->theta;
    if (!isfinite(theta)) return false;
    double first = 0.0, last = 0.0;
    out.magnitude = 1.0;
    if (kind == TQ_HIP_ROPE_YARN) {
        // the pair that makes so many turns over the trained length
        auto pair_of = [&](double turns) { return R * log(r->trained_len / (2.0 * pi * turns)) / (2.0 * log(theta)); };
        first = std::max(floor(pair_of(r->high)), 0.0);
        last = std::min(ceil(pair_of(r->low)), R - 1.0);
        out.magnitude = r->magnitude > 0.0 ? r->magnitude : 0.1 * log(s) + 1.0;
    }
    out.pairs = R / 2;
    for (int i = 0; i < out.pairs; i++) {
        double f = pow(theta, -2.0 * i / R);
        if (kind == TQ_HIP_ROPE_LINEAR) f /= s;
        if (kind == TQ_HIP_ROPE_BANDS) {
            const double turns = r->trained_len * f / (2.0 * pi);
            const double share = std::min(std::max((turns - r->low) / (r->high - r->low), 0.0), 1.0);
            f = f * share + f / s * (1.0 - share);
        }
        if (kind == TQ_HIP_ROPE_YARN) {
            const double ramp = std::min(std::max((i - first) / std::max(last - first, 0.001), 0.0), 1.0);
            f = f * (1.0 - ramp) + f / s * ramp;
        }
        out.f[i] = f;
    }
    return true;
}

bool heads_ok(const tq_hip_heads &t, int head_dim) {
    if (t.heads < 0 || t.heads > 65536) return false;
    if (t.heads == 0) return true;
    if (!t.x || !t.out || (((uintptr_t)t.x | (uintptr_t)t.out | (uintptr_t)t.norm) & 3)) return false;
    const size_t row = (size_t)t.heads * head_dim;
    if (t.stride < row || t.out_stride < row) return false;
    return t.out != t.x || t.out_stride == t.stride;
}

template <int LANES, int U>
void launch_norm_rope(const NormRopeArgs &a, int interleaved, int n, hipStream_t s) {
    constexpr int PER = 256 / LANES * U;
    const dim3 grid((unsigned)n, (unsigned)((a.heads + PER - 1) / PER));
    if (a.rot % (interleaved ? 4 : 8))
        hipLaunchKernelGGL((norm_rope_kernel<LANES, U, kAny>), grid, dim3(256), 0, s, a, interleaved);
    else if (interleaved)
        hipLaunchKernelGGL((norm_rope_kernel<LANES, U, kNeighbours>), grid, dim3(256), 0, s, a, interleaved);
    else
        hipLaunchKernelGGL((norm_rope_kernel<LANES, U, kHalves>), grid, dim3(256), 0, s, a, interleaved);
}

template <int LANES>
void launch_norm_rope(const NormRopeArgs &a, int interleaved, int n, hipStream_t s) {
    // up to four heads in flight per lane where that leaves work-groups enough for the
    // CUs, and a row's work-groups with equally many (8,192 rows of 72 heads of 128: three
    // 124 us, four 125 with lanes that have none, two 130, one 146)
    const int sets = (a.heads + 256 / LANES - 1) / (256 / LANES), wgs = (sets + 3) / 4;
    switch ((long)n * wgs >= 1024 ? (sets + wgs - 1) / wgs : 1) {
        case 1: return launch_norm_rope<LANES, 1>(a, interleaved, n, s);
        case 2: return launch_norm_rope<LANES, 2>(a, interleaved, n, s);
        case 3: return launch_norm_rope<LANES, 3>(a, interleaved, n, s);
        default: return launch_norm_rope<LANES, 4>(a, interleaved, n, s);
    }
}

int herr(hipError_t e) { return e == hipSuccess ? TQ_HIP_OK : TQ_HIP_EHIP_BASE - (int)e; }

}  // namespace

extern "C" {

int tq_hip_rope_rows(const tq_hip_rope *rope, int n, const int32_t *d_pos, float *d_cos, float *d_sin, void *stream) {
    Frequencies f;
    if (n < 0 || !frequencies(rope, f)) return TQ_HIP_EINVAL;
    if (n == 0) return TQ_HIP_OK;
    if (!d_cos || !d_sin || (((uintptr_t)d_pos | (uintptr_t)d_cos | (uintptr_t)d_sin) & 3)) return TQ_HIP_EINVAL;
    if ((size_t)n * rope->rotary_dim > (size_t)1 << 33) return TQ_HIP_EINVAL;   // threads of a launch
    const size_t total = (size_t)n * f.pairs, wgs = (total + 1023) / 1024;
    hipLaunchKernelGGL(rope_rows_kernel, dim3((unsigned)wgs), dim3(256), 0, (hipStream_t)stream, f, d_pos, total, d_cos,
                       d_sin);
    return herr(hipGetLastError());
}

int tq_hip_norm_rope(const tq_hip_rope *rope, int head_dim, int n, const int32_t *d_pos, const tq_hip_heads *q,
                     const tq_hip_heads *k, float eps, void *stream) {
    NormRopeArgs a;
    if (n < 0 || n > 1 << 23 || head_dim < 4 || head_dim % 4 || head_dim > 256 || !frequencies(rope, a.freq)) return TQ_HIP_EINVAL;
    if (rope->rotary_dim > head_dim || (uintptr_t)d_pos & 3) return TQ_HIP_EINVAL;
    a.q = q ? *q : tq_hip_heads{};
    a.k = k ? *k : tq_hip_heads{};
    if (!heads_ok(a.q, head_dim) || !heads_ok(a.k, head_dim)) return TQ_HIP_EINVAL;
    a.heads = a.q.heads + a.k.heads;
    if (n == 0 || a.heads == 0) return TQ_HIP_OK;
    a.pos = d_pos;
    a.head_dim = head_dim;
    a.rot = rope->rotary_dim;
    a.eps = eps;
    const int interleaved = rope->layout == TQ_HIP_ROPE_INTERLEAVED;
    const hipStream_t s = (hipStream_t)stream;
    if (head_dim <= 32)
        launch_norm_rope<8>(a, interleaved, n, s);
    else if (head_dim <= 64)
        launch_norm_rope<16>(a, interleaved, n, s);
    else if (head_dim <= 128)
        launch_norm_rope<32>(a, interleaved, n, s);
    else
        launch_norm_rope<64>(a, interleaved, n, s);
    return herr(hipGetLastError());
}

}  // extern "C"
