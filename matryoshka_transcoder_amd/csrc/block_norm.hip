// The norms before and after a block of a language model, fused with the block's gate and the residual add:
//     hidden = residual_scale * residual + branch_scale * gate * post(branch)          (post: none, RMS or layer norm)
//     normed = pre(hidden)                                                              (pre: RMS or layer norm)
//     norm(x) = u * (offset + w) + b,   u = (x - mu) * rstd,   mu = 0 for the RMS norm, rstd = 1 / sqrt(mean((x-mu)^2) + eps)
// and the gradient of all of it.  A transcoder that stands in for a model's MLP sits between the two (splice.py).
//
// Everything here is bound by memory: forward reads residual and branch and writes hidden and normed once, backward
// reads residual, branch and the two incoming gradients and writes two gradients.  hidden is NOT read back: it is
// recomputed from residual and branch, which costs the same bytes as reading it would and keeps its fp32 value (so the
// statistics, and the gradients through them, belong to the sum before its rounding to the model dtype).
//
// Layout: thread t of a row's T = 64 * ceil(A / 512) threads owns 8 columns for the whole launch, so the norm weights,
// the channel gate and the column sums of the weight gradients live in its registers while it walks over rows.  A
// workgroup holds `groups` such row groups.  Row sums: DPP inside a wave, one LDS exchange across the row's waves.
// Rows whose width is a multiple of 8 with 16-byte-aligned rows use 16-byte accesses (columns 8 t .. 8 t + 7); any other
// width or stride takes the same kernel with single elements (columns t, t + T, ..., which keeps a wave's accesses side by side).
#include "common.hpp"

namespace mtc {

constexpr int NORM_MAX_A = 8192;         // 1024 threads of 8 columns
constexpr int NORM_CUS = 256;            // MI355X: 256 CUs

struct NormRow {                         // one row-major operand: base, row stride in elements
    void* p;
    long long ld;
};

struct NormArgs {
    long long rows;
    int A, T, groups;
    int post_kind, pre_kind, gate_kind;
    float post_eps, pre_eps, post_off, pre_off, res_scale, branch_scale, inv_A;
    NormRow residual, branch, gate, hidden, normed;
    const void *post_w, *post_b, *pre_w, *pre_b;
    float* stats;                        // [4][rows]: post mean, post rstd, pre mean, pre rstd
    // backward
    NormRow d_hidden, d_normed;
    void *d_residual, *d_branch, *d_gate;
    float* partial;                      // [workgroup][4 vectors of `pitch` floats, then the scalar gate's sum]
    int pitch, want_x1, want_x2, want_x3, want_x4, want_scalar;
};

// sum over the 64 lanes, on DPP (six dependent VALU adds; the ds_bpermute form pays an LDS round trip per step)
template <int CTRL, int ROWS> __device__ __forceinline__ float dpp_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float row16_sum_at15(float v) {      // lane 15 of every 16 holds the sum of its 16
    v = dpp_add<0x111, 0xf>(v);
    v = dpp_add<0x112, 0xf>(v);
    v = dpp_add<0x114, 0xf>(v);
    return dpp_add<0x118, 0xf>(v);
}
__device__ __forceinline__ float lane_value(float v, int lane) {
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}
__device__ __forceinline__ float wave_total(float v) {
    v = row16_sum_at15(v);
    v = dpp_add<0x142, 0xa>(v);
    v = dpp_add<0x143, 0xc>(v);
    return lane_value(v, 63);
}

// Sums of N values over a row group.  Every wave of the workgroup calls it equally often; `slot` alternates between two
// LDS buffers, so one barrier per call orders the writes and the next call's writes cannot overtake this call's reads.
template <int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float* sm, int& slot, int group, int waves) {
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = wave_total(v[n]);
    if (waves == 1) return;
    const int lane = threadIdx.x & 63, wave = (int)(threadIdx.x >> 6) - group * waves;
    float* s = sm + slot * 16 * 4 + group * waves * 4;        // [2][16 waves of the workgroup][4 values]
    slot ^= 1;
    if (lane == 0) {
#pragma unroll
        for (int n = 0; n < N; ++n) s[wave * 4 + n] = v[n];
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = lane_value(row16_sum_at15(lane < waves ? s[(lane & 15) * 4 + n] : 0.f), 15);
}

// the 8 columns of thread t
template <int DT, bool VEC> struct Cols {
    int t, T, A;
    __device__ __forceinline__ int col(int i) const { return VEC ? t * 8 + i : t + T * i; }
    __device__ __forceinline__ bool in(int i) const { return VEC ? t * 8 < A : t + T * i < A; }
    // elements outside the row read as zero
    __device__ __forceinline__ void load(const void* base, long long off, float (&v)[8]) const {
        typedef typename DType<DT>::T T_;
        if (VEC) {
            if (in(0)) load8<DT>(base, (size_t)(off + t * 8), v);
            else
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = 0.f;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = in(i) ? DType<DT>::ld(reinterpret_cast<const T_*>(base) + off + col(i)) : 0.f;
        }
    }
    __device__ __forceinline__ void store(void* base, long long off, const float (&v)[8]) const {
        typedef typename DType<DT>::T T_;
        if (VEC) {
            if (in(0)) store8<DT>(base, (size_t)(off + t * 8), v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (in(i)) DType<DT>::st(reinterpret_cast<T_*>(base) + off + col(i), v[i]);
        }
    }
    // offset + w, or 1 without a weight; 0 outside the row
    __device__ __forceinline__ void weight(const void* w, float offset, float (&v)[8]) const {
        if (w) load(w, 0, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = in(i) ? (w ? offset + v[i] : 1.f) : 0.f;
    }
    __device__ __forceinline__ void bias(const void* b, float (&v)[8]) const {
        if (b) load(b, 0, v);
        else
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = 0.f;
    }
};

// mean and 1/std of a row held in registers: v becomes u.  The variance is summed over v - mu (not as E[x^2] - mu^2,
// which cancels for rows far from zero).
template <int DT, bool VEC>
__device__ __forceinline__ void normalise(const Cols<DT, VEC>& c, int kind, float eps, float inv_A, float (&v)[8], float* sm,
                                          int& slot, int group, int waves, float& mu, float& rstd) {
    mu = 0.f;
    if (kind == MTC_NORM_LAYER) {
        float s[1] = {0.f};
#pragma unroll
        for (int i = 0; i < 8; ++i) s[0] += v[i];
        group_sum(s, sm, slot, group, waves);
        mu = s[0] * inv_A;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = c.in(i) ? v[i] - mu : 0.f;
    }
    float q[1] = {0.f};
#pragma unroll
    for (int i = 0; i < 8; ++i) q[0] = fmaf(v[i], v[i], q[0]);
    group_sum(q, sm, slot, group, waves);
    rstd = 1.f / sqrtf(fmaf(q[0], inv_A, eps));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= rstd;
}

// factor and bias of the branch before the row / element gate: z = u_p * pf + pb
template <int DT, bool VEC>
__device__ __forceinline__ void branch_factors(const Cols<DT, VEC>& c, const NormArgs& a, float (&pf)[8], float (&pb)[8]) {
    c.weight(a.post_kind == MTC_NORM_NONE ? nullptr : a.post_w, a.post_off, pf);
    c.bias(a.post_kind == MTC_NORM_NONE ? nullptr : a.post_b, pb);
    float cg[8];
    if (a.gate_kind == MTC_GATE_CHANNEL) c.load(a.gate.p, 0, cg);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float s = a.gate_kind == MTC_GATE_CHANNEL ? a.branch_scale * cg[i] : a.branch_scale;
        pf[i] *= s;
        pb[i] *= s;
    }
}

template <int DT, bool VEC, bool BRANCH, bool PRE>
__global__ __launch_bounds__(1024) void block_norm_fwd_kernel(NormArgs a) {
    typedef typename DType<DT>::T T_;
    __shared__ float sm[2 * 16 * 4];
    const int waves = a.T >> 6;
    const int group = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6) / waves);
    const Cols<DT, VEC> c = {(int)threadIdx.x - group * a.T, a.T, a.A};
    int slot = 0;
    float pf[8], pb[8], qw[8], qb[8];
    if (BRANCH) branch_factors(c, a, pf, pb);
    if (PRE) { c.weight(a.pre_w, a.pre_off, qw); c.bias(a.pre_b, qb); }
    for (long long base = (long long)blockIdx.x * a.groups; base < a.rows; base += (long long)gridDim.x * a.groups) {
        const bool live = base + group < a.rows;
        const long long row = live ? base + group : a.rows - 1;       // groups behind the last row repeat it and store nothing
        float h[8];
        c.load(a.residual.p, row * a.residual.ld, h);
        if (BRANCH) {
            float y[8], g[8], gr = 1.f, mu = 0.f, rstd = 1.f;
            c.load(a.branch.p, row * a.branch.ld, y);
            if (a.gate_kind == MTC_GATE_FULL) c.load(a.gate.p, row * a.gate.ld, g);
            if (a.gate_kind == MTC_GATE_ROW || a.gate_kind == MTC_GATE_SCALAR)
                gr = DType<DT>::ld(reinterpret_cast<const T_*>(a.gate.p) + row * a.gate.ld);       // scalar: ld = 0
            if (a.post_kind != MTC_NORM_NONE) {
                normalise(c, a.post_kind, a.post_eps, a.inv_A, y, sm, slot, group, waves, mu, rstd);
                if (a.stats && live && c.t == 0) { a.stats[row] = mu; a.stats[a.rows + row] = rstd; }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float z = fmaf(y[i], pf[i], pb[i]);
                h[i] = fmaf(a.gate_kind == MTC_GATE_FULL ? g[i] : gr, z, a.res_scale * h[i]);
            }
            if (live) c.store(a.hidden.p, row * a.hidden.ld, h);
        }
        if (PRE) {
            float mu, rstd;
            normalise(c, a.pre_kind, a.pre_eps, a.inv_A, h, sm, slot, group, waves, mu, rstd);
            if (a.stats && live && c.t == 0) { a.stats[2 * a.rows + row] = mu; a.stats[3 * a.rows + row] = rstd; }
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = fmaf(h[i], qw[i], qb[i]);
            if (live) c.store(a.normed.p, row * a.normed.ld, h);
        }
    }
}

// Gradient.  With g = d_normed, du = g (offset + w_pre):
//     D        = d_hidden + rstd (du - [layer] mean(du) - u mean(du u))          d_residual = residual_scale D
//     dv       = D gate pf                                                       (pf: branch scale x channel gate x post weight)
//     d_branch = rstd_p (dv - [layer] mean(dv) - u_p mean(dv u_p))               (post norm; else dv)
// and the column sums (over rows) X1 = gate D u_p, X2 = gate D, X3 = g u, X4 = g, from which block_norm_cols_kernel makes the
// gradients of the weights, biases and the channel gate.  Each workgroup leaves one partial per column, summed in a
// fixed order afterwards: no atomics, the same bits on every run.
template <int DT, bool VEC, bool BRANCH, bool PRE, int SUMS /* 0 none, 1 X1 X3, 2 all */>
__global__ __launch_bounds__(1024) void block_norm_bwd_kernel(NormArgs a) {
    typedef typename DType<DT>::T T_;
    __shared__ float sm[2 * 16 * 4];
    extern __shared__ float fold[];                      // (groups - 1) * T * 8 floats when SUMS > 0
    const int waves = a.T >> 6;
    const int group = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6) / waves);
    const Cols<DT, VEC> c = {(int)threadIdx.x - group * a.T, a.T, a.A};
    int slot = 0;
    float pf[8], pb[8], qw[8];
    float x1[8], x2[8], x3[8], x4[8], gate_sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) x1[i] = x2[i] = x3[i] = x4[i] = 0.f;
    if (BRANCH) branch_factors(c, a, pf, pb);
    if (PRE) c.weight(a.pre_w, a.pre_off, qw);
    for (long long base = (long long)blockIdx.x * a.groups; base < a.rows; base += (long long)gridDim.x * a.groups) {
        const bool live = base + group < a.rows;
        const long long row = live ? base + group : a.rows - 1;
        float D[8], up[8], z[8], g[8], gr = 1.f, rstd_p = 1.f;
        if (BRANCH) {
            c.load(a.branch.p, row * a.branch.ld, up);
            if (a.gate_kind == MTC_GATE_FULL) c.load(a.gate.p, row * a.gate.ld, g);
            if (a.gate_kind == MTC_GATE_ROW || a.gate_kind == MTC_GATE_SCALAR)
                gr = DType<DT>::ld(reinterpret_cast<const T_*>(a.gate.p) + row * a.gate.ld);       // scalar: ld = 0
            if (a.post_kind != MTC_NORM_NONE) {
                const float mu_p = a.stats[row];
                rstd_p = a.stats[a.rows + row];
#pragma unroll
                for (int i = 0; i < 8; ++i) up[i] = (up[i] - mu_p) * rstd_p;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) z[i] = fmaf(up[i], pf[i], pb[i]);
            if (a.gate_kind != MTC_GATE_FULL)
#pragma unroll
                for (int i = 0; i < 8; ++i) g[i] = gr;
            if (a.d_hidden.p) c.load(a.d_hidden.p, row * a.d_hidden.ld, D);
        }
        if (!BRANCH || !a.d_hidden.p)
#pragma unroll
            for (int i = 0; i < 8; ++i) D[i] = 0.f;
        if (PRE) {
            float u[8], dn[8];
            c.load(a.residual.p, row * a.residual.ld, u);
            c.load(a.d_normed.p, row * a.d_normed.ld, dn);
            const float mu = a.stats[2 * a.rows + row], rstd = a.stats[3 * a.rows + row];
            float s[2] = {0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (BRANCH) u[i] = fmaf(g[i], z[i], a.res_scale * u[i]);
                u[i] = (u[i] - mu) * rstd;
                if (SUMS >= 1 && live) x3[i] = fmaf(dn[i], u[i], x3[i]);
                if (SUMS >= 2 && live) x4[i] += dn[i];
                dn[i] *= qw[i];
                s[0] += dn[i];
                s[1] = fmaf(dn[i], u[i], s[1]);
            }
            group_sum(s, sm, slot, group, waves);
            const float m1 = a.pre_kind == MTC_NORM_LAYER ? s[0] * a.inv_A : 0.f, m2 = s[1] * a.inv_A;
#pragma unroll
            for (int i = 0; i < 8; ++i) D[i] = fmaf(rstd, dn[i] - m1 - u[i] * m2, D[i]);
        }
        if (a.d_residual && live) {
            float o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = BRANCH ? a.res_scale * D[i] : D[i];
            c.store(a.d_residual, row * a.A, o);
        }
        if (BRANCH) {
            float s[3] = {0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                z[i] *= D[i];                            // d gate, before its reduction
                s[2] += z[i];
            }
            if (a.gate_kind == MTC_GATE_FULL && a.d_gate && live) c.store(a.d_gate, row * a.A, z);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                D[i] *= g[i];
                if (SUMS >= 1 && live) x1[i] = fmaf(D[i], up[i], x1[i]);
                if (SUMS >= 2 && live) x2[i] += D[i];
                D[i] *= pf[i];
                s[0] += D[i];
                s[1] = fmaf(D[i], up[i], s[1]);
            }
            const bool row_gate = a.gate_kind == MTC_GATE_ROW && a.d_gate;
            if (a.post_kind != MTC_NORM_NONE || row_gate || a.want_scalar) {
                group_sum(s, sm, slot, group, waves);
                if (row_gate && live && c.t == 0) DType<DT>::st(reinterpret_cast<T_*>(a.d_gate) + row, s[2]);
                if (live) gate_sum += s[2];
            }
            if (a.d_branch && live) {
                if (a.post_kind != MTC_NORM_NONE) {
                    const float m1 = a.post_kind == MTC_NORM_LAYER ? s[0] * a.inv_A : 0.f, m2 = s[1] * a.inv_A;
#pragma unroll
                    for (int i = 0; i < 8; ++i) D[i] = rstd_p * (D[i] - m1 - up[i] * m2);
                }
                c.store(a.d_branch, row * a.A, D);
            }
        }
    }
    if constexpr (SUMS > 0) {
        // the groups' column sums folded through LDS, one partial per workgroup (vectors nobody asked for are skipped)
        float* out = a.partial + (size_t)blockIdx.x * (4 * a.pitch + 8);
        if (a.want_scalar) {
            __syncthreads();
            if (c.t == 0) sm[group] = gate_sum;
            __syncthreads();
            if (threadIdx.x == 0) {
                for (int q = 1; q < a.groups; ++q) gate_sum += sm[q];
                out[4 * a.pitch] = gate_sum;
            }
        }
        auto put = [&](float (&x)[8], int want, int which) {
            if (!want) return;                           // the same for the whole launch
            __syncthreads();
            if (group > 0)
#pragma unroll
                for (int i = 0; i < 8; ++i) fold[((group - 1) * 8 + i) * a.T + c.t] = x[i];
            __syncthreads();
            if (group == 0) {
                for (int q = 1; q < a.groups; ++q)
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] += fold[((q - 1) * 8 + i) * a.T + c.t];
                Cols<MTC_F32, VEC>{c.t, c.T, c.A}.store(out + (size_t)which * a.pitch, 0, x);
            }
        };
        put(x1, a.want_x1, 0);
        if (SUMS >= 2) put(x2, a.want_x2, 1);
        put(x3, a.want_x3, 2);
        if (SUMS >= 2) put(x4, a.want_x4, 3);
    }
}

struct NormCols {
    int A, parts, pitch, gate_kind;
    float branch_scale, post_off;
    const float* partial;
    const void *gate, *post_w, *post_b;      // gate: the channel gate, else unused; post_w / post_b may be NULL
    void *d_post_w, *d_post_b, *d_gate, *d_pre_w, *d_pre_b;
    int want_x1, want_x2, want_scalar;
};

// the last sums over the workgroups' partials: 64 columns per workgroup, its 16 waves share the partials
template <int DT>
__global__ __launch_bounds__(1024) void block_norm_cols_kernel(NormCols n) {
    typedef typename DType<DT>::T T_;
    __shared__ float sm[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = blockIdx.x * 64 + lane;
    auto total = [&](int which) {
        float s = 0.f;
        if (col < n.A) {
            const float* p = n.partial + (size_t)which * n.pitch + col;
#pragma unroll 8
            for (int i = wave; i < n.parts; i += 16) s += p[(size_t)i * (4 * n.pitch + 8)];
        }
        __syncthreads();
        sm[wave][lane] = s;
        __syncthreads();
        s = 0.f;
#pragma unroll
        for (int w = 0; w < 16; ++w) s += sm[w][lane];
        return s;
    };
    auto put = [&](void* out, float v) {
        if (out && wave == 0 && col < n.A) DType<DT>::st(reinterpret_cast<T_*>(out) + col, v);
    };
    auto get = [&](const void* p) { return DType<DT>::ld(reinterpret_cast<const T_*>(p) + col); };
    if (blockIdx.y == 0) {
        if (n.want_scalar && blockIdx.x == 0 && wave == 0) {
            float s = 0.f;
            for (int i = lane; i < n.parts; i += 64) s += n.partial[(size_t)i * (4 * n.pitch + 8) + 4 * n.pitch];
            s = wave_total(s);
            if (lane == 0) DType<DT>::st(reinterpret_cast<T_*>(n.d_gate), s);
        }
        const float x1 = n.want_x1 ? total(0) : 0.f, x2 = n.want_x2 ? total(1) : 0.f;
        if (col >= n.A) return;
        const float s = n.branch_scale * (n.gate_kind == MTC_GATE_CHANNEL ? get(n.gate) : 1.f);
        put(n.d_post_w, s * x1);
        put(n.d_post_b, s * x2);
        if (n.gate_kind == MTC_GATE_CHANNEL && n.d_gate) {
            const float w = n.post_w ? n.post_off + get(n.post_w) : 1.f, b = n.post_b ? get(n.post_b) : 0.f;
            put(n.d_gate, n.branch_scale * (w * x1 + b * x2));
        }
    } else {
        if (n.d_pre_w) put(n.d_pre_w, total(2));
        if (n.d_pre_b) put(n.d_pre_b, total(3));
    }
}

}  // namespace mtc

using namespace mtc;

static int norm_check(const mtc_block_norm_desc* d, const char* who) {
    MTC_REQUIRE(d, "%s: null descriptor", who);
    MTC_REQUIRE(d->dtype == MTC_F32 || d->dtype == MTC_BF16, "%s: bad dtype %d", who, d->dtype);
    MTC_REQUIRE(d->A >= 1 && d->A <= NORM_MAX_A, "%s: width %d outside 1..%d", who, d->A, NORM_MAX_A);
    MTC_REQUIRE(d->rows >= 0 && d->rows < (1ll << 40), "%s: bad row count %lld", who, (long long)d->rows);
    auto kind_ok = [](int k) { return k == MTC_NORM_NONE || k == MTC_NORM_RMS || k == MTC_NORM_LAYER; };
    MTC_REQUIRE(kind_ok(d->post_kind) && kind_ok(d->pre_kind), "%s: bad norm kind (%d, %d)", who, d->post_kind, d->pre_kind);
    MTC_REQUIRE(d->gate_kind >= MTC_GATE_NONE && d->gate_kind <= MTC_GATE_SCALAR, "%s: bad gate kind %d", who, d->gate_kind);
    MTC_REQUIRE(d->has_branch || d->pre_kind != MTC_NORM_NONE, "%s: neither a branch nor a norm", who);
    MTC_REQUIRE(d->has_branch || (d->post_kind == MTC_NORM_NONE && d->gate_kind == MTC_GATE_NONE && d->residual_scale == 1.f),
                "%s: post norm, gate and residual scale need a branch", who);
    MTC_REQUIRE(d->ld_residual >= 0 && d->ld_branch >= 0 && d->ld_gate >= 0 && d->ld_hidden >= 0 && d->ld_normed >= 0,
                "%s: negative row stride", who);
    return 0;
}

static int norm_threads(int A) { return ((A + 7) / 8 + 63) / 64 * 64; }

static int norm_elem(int dtype) { return dtype == MTC_BF16 ? 2 : 4; }

static bool row_vec(const void* p, long long ld, long long rows, int dtype) {
    return !p || (((uintptr_t)p & 15) == 0 && (rows <= 1 || ((ld * norm_elem(dtype)) & 15) == 0));
}

static void norm_args(const mtc_block_norm_desc* d, NormArgs& a) {
    a = NormArgs{};
    a.rows = d->rows; a.A = d->A; a.T = norm_threads(d->A);
    a.post_kind = d->post_kind; a.pre_kind = d->pre_kind; a.gate_kind = d->gate_kind;
    a.post_eps = d->post_eps; a.pre_eps = d->pre_eps; a.post_off = d->post_offset; a.pre_off = d->pre_offset;
    a.res_scale = d->residual_scale; a.branch_scale = d->branch_scale;
    a.inv_A = 1.f / (float)d->A;
}

static int norm_operands(const mtc_block_norm_desc* d, const char* who, const void* residual, const void* branch, const void* gate,
                         NormArgs& a) {
    MTC_REQUIRE(residual, "%s: null residual", who);
    MTC_REQUIRE(!d->has_branch == !branch, "%s: branch pointer and has_branch disagree", who);
    MTC_REQUIRE((d->gate_kind == MTC_GATE_NONE) == !gate, "%s: gate pointer and gate_kind disagree", who);
    a.residual = {const_cast<void*>(residual), d->ld_residual};
    a.branch = {const_cast<void*>(branch), d->ld_branch};
    a.gate = {const_cast<void*>(gate), d->gate_kind == MTC_GATE_SCALAR ? 0 : d->ld_gate};
    return 0;
}

static bool norm_inputs_vec(const mtc_block_norm_desc* d, const NormArgs& a) {
    return (d->A & 7) == 0 && row_vec(a.residual.p, a.residual.ld, d->rows, d->dtype) &&
           row_vec(a.branch.p, a.branch.ld, d->rows, d->dtype) &&
           ((a.gate_kind != MTC_GATE_CHANNEL && a.gate_kind != MTC_GATE_FULL) ||
            row_vec(a.gate.p, a.gate_kind == MTC_GATE_FULL ? a.gate.ld : 0, d->rows, d->dtype)) &&
           row_vec(a.post_w, 0, 1, d->dtype) && row_vec(a.post_b, 0, 1, d->dtype) && row_vec(a.pre_w, 0, 1, d->dtype) &&
           row_vec(a.pre_b, 0, 1, d->dtype);
}

template <int DT, bool VEC> static void launch_norm_fwd(const NormArgs& a, bool branch, unsigned grid, hipStream_t s) {
    const dim3 b(a.T * a.groups);
    if (branch && a.pre_kind != MTC_NORM_NONE) hipLaunchKernelGGL((block_norm_fwd_kernel<DT, VEC, true, true>), dim3(grid), b, 0, s, a);
    else if (branch) hipLaunchKernelGGL((block_norm_fwd_kernel<DT, VEC, true, false>), dim3(grid), b, 0, s, a);
    else hipLaunchKernelGGL((block_norm_fwd_kernel<DT, VEC, false, true>), dim3(grid), b, 0, s, a);
}

extern "C" int mtc_block_norm_fwd(const mtc_block_norm_desc* d, const void* residual, const void* branch, const void* gate,
                                  const void* post_w, const void* post_b, const void* pre_w, const void* pre_b, void* hidden,
                                  void* normed, float* stats, void* stream) {
    static const char* who = "mtc_block_norm_fwd";
    if (norm_check(d, who)) return -1;
    if (d->rows == 0) return 0;
    NormArgs a;
    norm_args(d, a);
    if (norm_operands(d, who, residual, branch, gate, a)) return -1;
    MTC_REQUIRE(!d->has_branch == !hidden, "%s: hidden is written exactly when there is a branch", who);
    MTC_REQUIRE((d->pre_kind == MTC_NORM_NONE) == !normed, "%s: normed pointer and pre_kind disagree", who);
    MTC_REQUIRE(d->rows <= 1 || ((!hidden || d->ld_hidden >= d->A) && (!normed || d->ld_normed >= d->A)),
                "%s: output rows overlap (row stride below the width)", who);
    a.hidden = {hidden, d->ld_hidden};
    a.normed = {normed, d->ld_normed};
    a.post_w = post_w; a.post_b = post_b; a.pre_w = pre_w; a.pre_b = pre_b;
    a.stats = stats;
    const bool vec = norm_inputs_vec(d, a) && row_vec(hidden, d->ld_hidden, d->rows, d->dtype) &&
                     row_vec(normed, d->ld_normed, d->rows, d->dtype);
    a.groups = a.T >= 256 ? 1 : 256 / a.T;
    const long long want = (d->rows + a.groups - 1) / a.groups;
    const unsigned grid = (unsigned)(want < NORM_CUS * 8 ? want : NORM_CUS * 8);
    hipStream_t s = as_stream(stream);
    if (d->dtype == MTC_BF16) vec ? launch_norm_fwd<MTC_BF16, true>(a, branch, grid, s) : launch_norm_fwd<MTC_BF16, false>(a, branch, grid, s);
    else vec ? launch_norm_fwd<MTC_F32, true>(a, branch, grid, s) : launch_norm_fwd<MTC_F32, false>(a, branch, grid, s);
    return check_launch(who);
}

// backward launch shape: one workgroup per CU of up to 1024 threads, fewer row groups when there are few rows
static void norm_bwd_shape(const mtc_block_norm_desc* d, int& groups, unsigned& grid) {
    const int T = norm_threads(d->A);
    const long long per_cu = (d->rows + NORM_CUS - 1) / NORM_CUS;
    groups = (int)(per_cu < 1024 / T ? per_cu : 1024 / T);
    if (groups < 1) groups = 1;
    const long long want = (d->rows + groups - 1) / groups;
    grid = (unsigned)(want < NORM_CUS ? want : NORM_CUS);
}

extern "C" size_t mtc_block_norm_bwd_workspace_bytes(const mtc_block_norm_desc* d) {
    if (norm_check(d, "mtc_block_norm_bwd_workspace_bytes")) return 0;
    if (d->rows == 0) return 0;
    int groups;
    unsigned grid;
    norm_bwd_shape(d, groups, grid);
    return (size_t)grid * (4 * ((d->A + 7) / 8 * 8) + 8) * sizeof(float);
}

template <int DT, bool VEC, bool BRANCH, bool PRE>
static void launch_norm_bwd(const NormArgs& a, int sums, unsigned grid, hipStream_t s) {
    const dim3 b(a.T * a.groups);
    const size_t lds = sums ? (size_t)(a.groups - 1) * a.T * 8 * sizeof(float) : 0;
    if (sums == 0) hipLaunchKernelGGL((block_norm_bwd_kernel<DT, VEC, BRANCH, PRE, 0>), dim3(grid), b, lds, s, a);
    else if (sums == 1) hipLaunchKernelGGL((block_norm_bwd_kernel<DT, VEC, BRANCH, PRE, 1>), dim3(grid), b, lds, s, a);
    else hipLaunchKernelGGL((block_norm_bwd_kernel<DT, VEC, BRANCH, PRE, 2>), dim3(grid), b, lds, s, a);
}

template <int DT, bool VEC> static void launch_norm_bwd_mode(const NormArgs& a, bool branch, int sums, unsigned grid, hipStream_t s) {
    if (branch && a.pre_kind != MTC_NORM_NONE) launch_norm_bwd<DT, VEC, true, true>(a, sums, grid, s);
    else if (branch) launch_norm_bwd<DT, VEC, true, false>(a, sums, grid, s);
    else launch_norm_bwd<DT, VEC, false, true>(a, sums, grid, s);
}

extern "C" int mtc_block_norm_bwd(const mtc_block_norm_desc* d, const void* residual, const void* branch, const void* gate,
                                  const void* post_w, const void* post_b, const void* pre_w, const void* pre_b,
                                  const float* stats, const void* d_hidden, int64_t ld_d_hidden, const void* d_normed,
                                  int64_t ld_d_normed, void* d_residual, void* d_branch, void* d_gate, void* d_post_w,
                                  void* d_post_b, void* d_pre_w, void* d_pre_b, void* workspace, size_t workspace_bytes,
                                  void* stream) {
    static const char* who = "mtc_block_norm_bwd";
    if (norm_check(d, who)) return -1;
    MTC_REQUIRE(d->rows > 0, "%s: no rows (the gradients of the weights are zero then: fill them)", who);
    NormArgs a;
    norm_args(d, a);
    if (norm_operands(d, who, residual, branch, gate, a)) return -1;
    MTC_REQUIRE((d->pre_kind == MTC_NORM_NONE) == !d_normed, "%s: d_normed pointer and pre_kind disagree", who);
    MTC_REQUIRE(d->has_branch || !(d_hidden || d_branch || d_gate || d_post_w || d_post_b), "%s: gradient of an absent branch", who);
    MTC_REQUIRE(d->pre_kind != MTC_NORM_NONE || !(d_pre_w || d_pre_b), "%s: gradient of an absent pre norm", who);
    MTC_REQUIRE(d->post_kind != MTC_NORM_NONE || !(d_post_w || d_post_b), "%s: gradient of an absent post norm", who);
    MTC_REQUIRE(d->gate_kind != MTC_GATE_NONE || !d_gate, "%s: gradient of an absent gate", who);
    MTC_REQUIRE(stats || (d->pre_kind == MTC_NORM_NONE && d->post_kind == MTC_NORM_NONE), "%s: null stats", who);
    MTC_REQUIRE(ld_d_hidden >= 0 && ld_d_normed >= 0, "%s: negative row stride", who);
    a.post_w = post_w; a.post_b = post_b; a.pre_w = pre_w; a.pre_b = pre_b;
    a.stats = const_cast<float*>(stats);
    a.d_hidden = {const_cast<void*>(d_hidden), ld_d_hidden};
    a.d_normed = {const_cast<void*>(d_normed), ld_d_normed};
    a.d_residual = d_residual; a.d_branch = d_branch; a.d_gate = d_gate;
    const bool chan = d->gate_kind == MTC_GATE_CHANNEL && d_gate;
    const bool chan_bias = chan && d->post_kind != MTC_NORM_NONE && post_b;
    a.want_x1 = d_post_w || chan;
    a.want_x2 = d_post_b || chan_bias;
    a.want_x3 = d_pre_w != nullptr;
    a.want_x4 = d_pre_b != nullptr;
    a.want_scalar = d->gate_kind == MTC_GATE_SCALAR && d_gate;
    const int sums = a.want_x2 || a.want_x4 ? 2 : a.want_x1 || a.want_x3 || a.want_scalar ? 1 : 0;
    a.pitch = (d->A + 7) / 8 * 8;
    unsigned grid;
    norm_bwd_shape(d, a.groups, grid);
    if (sums) {
        MTC_REQUIRE(workspace && workspace_bytes >= mtc_block_norm_bwd_workspace_bytes(d), "%s: workspace too small", who);
        MTC_REQUIRE(((uintptr_t)workspace & 15) == 0, "%s: workspace must be 16-byte aligned", who);
        a.partial = reinterpret_cast<float*>(workspace);
    }
    const long long A = d->A;
    const bool vec = norm_inputs_vec(d, a) && row_vec(d_hidden, ld_d_hidden, d->rows, d->dtype) &&
                     row_vec(d_normed, ld_d_normed, d->rows, d->dtype) && row_vec(d_residual, A, d->rows, d->dtype) &&
                     row_vec(d_branch, A, d->rows, d->dtype) &&
                     (d->gate_kind != MTC_GATE_FULL || row_vec(d_gate, A, d->rows, d->dtype));
    hipStream_t s = as_stream(stream);
    if (d->dtype == MTC_BF16)
        vec ? launch_norm_bwd_mode<MTC_BF16, true>(a, branch, sums, grid, s) : launch_norm_bwd_mode<MTC_BF16, false>(a, branch, sums, grid, s);
    else
        vec ? launch_norm_bwd_mode<MTC_F32, true>(a, branch, sums, grid, s) : launch_norm_bwd_mode<MTC_F32, false>(a, branch, sums, grid, s);
    if (check_launch(who)) return -2;
    if (sums) {
        NormCols n = {};
        n.A = d->A; n.parts = (int)grid; n.pitch = a.pitch; n.gate_kind = d->gate_kind;
        n.branch_scale = d->branch_scale; n.post_off = d->post_offset;
        n.partial = a.partial;
        n.gate = gate;
        n.post_w = d->post_kind == MTC_NORM_NONE ? nullptr : post_w;
        n.post_b = d->post_kind == MTC_NORM_NONE ? nullptr : post_b;
        n.d_post_w = d_post_w; n.d_post_b = d_post_b; n.d_gate = chan || a.want_scalar ? d_gate : nullptr;
        n.d_pre_w = d_pre_w; n.d_pre_b = d_pre_b;
        n.want_x1 = a.want_x1; n.want_x2 = a.want_x2; n.want_scalar = a.want_scalar;
        const dim3 g2((d->A + 63) / 64, 2);
        if (d->dtype == MTC_BF16) hipLaunchKernelGGL(block_norm_cols_kernel<MTC_BF16>, g2, dim3(1024), 0, s, n);
        else hipLaunchKernelGGL(block_norm_cols_kernel<MTC_F32>, g2, dim3(1024), 0, s, n);
        return check_launch(who);
    }
    return 0;
}
