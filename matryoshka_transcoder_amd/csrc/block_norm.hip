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
// Rows of a multiple of 16 bytes that start at multiples of 16 bytes use 16-byte accesses (columns 8 t .. 8 t + 7); any other
// width or stride takes the same kernel with single elements (columns t, t + T, ..., which keeps a wave's accesses side by side).
#include <algorithm>
#include <type_traits>
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
    int post_kind, pre_kind, gate_kind, streaming;
    float post_eps, pre_eps, post_off, pre_off, res_scale, branch_scale, inv_A;
    NormRow residual, branch, gate, hidden, normed;
    const void *post_w, *post_b, *pre_w, *pre_b;
    float* stats;                        // [rows][4]: post mean, post rstd, pre mean, pre rstd
    // backward
    NormRow d_hidden, d_normed, d_residual, d_branch, d_gate;
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

// Rows are read and written through buffer instructions: a descriptor per row (built in scalar registers) whose size is the
// row's, so that threads beyond the width read zeros and write nothing WITHOUT a branch.  Branches around the memory
// instructions made the compiler wait for every load in flight at each join, which undid the prefetch below (a row's
// loads then cost their full latency: 16384 x 4608 bf16, pair: forward 148 instead of 118 us, backward 329 instead of 178).
typedef __amdgpu_buffer_rsrc_t rsrc_t;
__device__ __forceinline__ rsrc_t rows_rsrc(const void* base, long long byte_off, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(reinterpret_cast<const char*>(base)) + byte_off, 0, bytes, 0x00020000);
}

// the 8 columns of thread t, and 8 values as they lie in memory: what a load in flight occupies
//   STREAM: non-temporal accesses, for passes over more than the Infinity Cache holds
template <int DT, bool VEC, bool STREAM> struct Cols {
    static constexpr int AUX = STREAM ? 2 : 0;
    typedef typename DType<DT>::T T_;
    static constexpr int ES = (int)sizeof(T_);
    static constexpr int NR = VEC ? 8 * ES / 16 : 8;
    struct Raw {
        typedef std::conditional_t<VEC, u32x4, T_> R;
        R r[NR];
        __device__ __forceinline__ void unpack(float (&v)[8]) const {
            if constexpr (VEC && DT == MTC_BF16) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[2 * i] = __uint_as_float(r[0][i] << 16);
                    v[2 * i + 1] = __uint_as_float(r[0][i] & 0xffff0000u);
                }
            } else if constexpr (VEC) {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i >> 2][i & 3]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = DType<DT>::ld(&r[i]);
            }
        }
    };
    int t, T, A;
    // bf16: 8 columns in a row; fp32: two runs of 4, T quads apart, so that every 16-byte access of a wave is contiguous
    __device__ __forceinline__ int col(int i) const {
        return !VEC ? t + T * i : ES == 2 ? t * 8 + i : (i < 4 ? t * 4 + i : (T + t) * 4 + i - 4);
    }
    __device__ __forceinline__ bool in(int i) const { return col(VEC ? i & ~(16 / ES - 1) : i) < A; }
    __device__ __forceinline__ void fetch(rsrc_t s, Raw& q) const {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < NR; ++i) q.r[i] = __builtin_amdgcn_raw_buffer_load_b128(s, col(i * (16 / ES)) * ES, 0, AUX);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if constexpr (ES == 2) q.r[i] = __builtin_amdgcn_raw_buffer_load_b16(s, col(i) * ES, 0, 0);
                else q.r[i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(s, col(i) * ES, 0, 0));
            }
        }
    }
    // `present` = false: zeros, and nothing is read
    __device__ __forceinline__ void fetch(const NormRow& o, long long row, bool present, Raw& q) const {
        fetch(rows_rsrc(o.p, row * o.ld * ES, present ? A * ES : 0), q);
    }
    __device__ __forceinline__ void store(rsrc_t s, const float (&v)[8]) const {
        if constexpr (VEC && DT == MTC_BF16) {
            u32x4 r;
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = pack2_bf16(v[2 * i], v[2 * i + 1]);
            __builtin_amdgcn_raw_buffer_store_b128(r, s, t * 8 * ES, 0, AUX);
        } else if constexpr (VEC) {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                u32x4 r;
#pragma unroll
                for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(v[4 * k + i]);
                __builtin_amdgcn_raw_buffer_store_b128(r, s, col(4 * k) * ES, 0, AUX);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if constexpr (ES == 2) __builtin_amdgcn_raw_buffer_store_b16((u16)f32_to_bf16_bits(v[i]), s, col(i) * ES, 0, 0);
                else __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v[i]), s, col(i) * ES, 0, 0);
            }
        }
    }
    __device__ __forceinline__ void store(const NormRow& o, long long row, bool present, const float (&v)[8]) const {
        store(rows_rsrc(o.p, row * o.ld * ES, present ? A * ES : 0), v);
    }
};

// mean and 1/std of a row held in registers: v becomes u.  The variance is summed over v - mu (not as E[x^2] - mu^2,
// which cancels for rows far from zero).
template <typename COLS>
__device__ __forceinline__ void normalise(const COLS& c, int kind, float eps, float inv_A, float (&v)[8], float* sm,
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

// The weights a thread keeps for the launch: the branch before the row / element gate is z = u_p * pf + pb, the pre norm
// u * qw + qb.  All loads go out before the first is waited for; an absent operand reads as zeros.
struct NormWeights {
    float pf[8], pb[8], qw[8], qb[8];
    template <typename COLS> __device__ __forceinline__ void load(const COLS& c, const NormArgs& a, bool branch, bool pre) {
        typename COLS::Raw w0, b0, g0, w1, b1;
        const bool post = branch && a.post_kind != MTC_NORM_NONE, chan = branch && a.gate_kind == MTC_GATE_CHANNEL;
        const bool pw = post && a.post_w, qw_ = pre && a.pre_w;
        if (branch) {
            c.fetch(NormRow{const_cast<void*>(a.post_w), 0}, 0, pw, w0);
            c.fetch(NormRow{const_cast<void*>(a.post_b), 0}, 0, post && a.post_b, b0);
            c.fetch(NormRow{a.gate.p, 0}, 0, chan, g0);
        }
        if (pre) {
            c.fetch(NormRow{const_cast<void*>(a.pre_w), 0}, 0, qw_, w1);
            c.fetch(NormRow{const_cast<void*>(a.pre_b), 0}, 0, a.pre_b != nullptr, b1);
        }
        if (branch) {
            float g[8];
            w0.unpack(pf);
            b0.unpack(pb);
            g0.unpack(g);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float s = c.in(i) ? (chan ? a.branch_scale * g[i] : a.branch_scale) : 0.f;
                pf[i] = s * (pw ? a.post_off + pf[i] : 1.f);
                pb[i] *= s;
            }
        }
        if (pre) {
            w1.unpack(qw);
            b1.unpack(qb);
#pragma unroll
            for (int i = 0; i < 8; ++i) qw[i] = c.in(i) ? (qw_ ? a.pre_off + qw[i] : 1.f) : 0.f;
        }
    }
};

// Walks a group's rows, two sets of operands in turn: while one row is computed, the next one's loads are in flight (the
// two sets have names of their own: moving a register that a load has yet to fill would wait for it).
template <bool PREFETCH, typename ROW, typename FETCH, typename COMPUTE>
__device__ __forceinline__ void walk_rows(long long base, long long step, long long rows, FETCH fetch, ROW& s0, COMPUTE compute) {
    if constexpr (!PREFETCH) {
        for (; base < rows; base += step) {
            compute(base, s0);
            if (base + step < rows) fetch(base + step, s0);
        }
    } else {
        ROW s1;
        while (base < rows) {
            fetch(base + step, s1);
            compute(base, s0);
            base += step;
            if (base >= rows) break;
            fetch(base + step, s0);
            compute(base, s1);
            base += step;
        }
    }
}

template <typename COLS, bool FULL> struct FwdRow {
    typename COLS::Raw residual, branch, gate[FULL ? 1 : 0];
    uint32_t gr;                         // the row's gate as it lies in memory
};

template <int DT> __device__ __forceinline__ uint32_t fetch_one(const NormRow& o, long long row, bool present) {
    constexpr int ES = (int)sizeof(typename DType<DT>::T);
    const rsrc_t s = rows_rsrc(o.p, row * o.ld * ES, present ? ES : 0);
    if constexpr (ES == 2) return (uint32_t)__builtin_amdgcn_raw_buffer_load_b16(s, 0, 0, 0) << 16;
    else return __builtin_amdgcn_raw_buffer_load_b32(s, 0, 0, 0);
}

template <int DT, bool VEC, bool BRANCH, bool PRE, bool FULL, bool STREAM>
__global__ __launch_bounds__(1024) void block_norm_fwd_kernel(NormArgs a) {
    __shared__ float sm[2 * 16 * 4];
    const int waves = a.T >> 6;
    const int group = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6) / waves);
    const Cols<DT, VEC, STREAM> c = {(int)threadIdx.x - group * a.T, a.T, a.A};
    int slot = 0;
    const bool row_gate = a.gate_kind == MTC_GATE_ROW || a.gate_kind == MTC_GATE_SCALAR;         // scalar: ld = 0
    const long long base0 = (long long)blockIdx.x * a.groups, step = (long long)gridDim.x * a.groups;
    typedef FwdRow<Cols<DT, VEC, STREAM>, FULL> Row;
    auto fetch = [&](long long base, Row& q) {
        const bool live = base + group < a.rows;
        const long long row = live ? base + group : 0;
        c.fetch(a.residual, row, live, q.residual);
        if (BRANCH) {
            c.fetch(a.branch, row, live, q.branch);
            if (FULL) c.fetch(a.gate, row, live, q.gate[0]);
            else q.gr = fetch_one<DT>(a.gate, row, live && row_gate);
        }
    };
    Row first;
    fetch(base0, first);
    NormWeights w;
    w.load(c, a, BRANCH, PRE);
    walk_rows<VEC>(base0, step, a.rows, fetch, first, [&](long long base, const Row& q) {
        const bool live = base + group < a.rows;                  // groups behind the last row compute on zeros and store nothing
        const long long row = live ? base + group : 0;
        float h[8], st[4] = {0.f, 0.f, 0.f, 0.f};
        q.residual.unpack(h);
        if (BRANCH) {
            float y[8], g[8];
            q.branch.unpack(y);
            if (FULL) q.gate[0].unpack(g);
            const float gr = row_gate ? __uint_as_float(q.gr) : 1.f;
            if (a.post_kind != MTC_NORM_NONE)
                normalise(c, a.post_kind, a.post_eps, a.inv_A, y, sm, slot, group, waves, st[0], st[1]);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = fmaf(FULL ? g[i] : gr, fmaf(y[i], w.pf[i], w.pb[i]), a.res_scale * h[i]);
            c.store(a.hidden, row, live, h);
        }
        if (PRE) {
            normalise(c, a.pre_kind, a.pre_eps, a.inv_A, h, sm, slot, group, waves, st[2], st[3]);
#pragma unroll
            for (int i = 0; i < 8; ++i) h[i] = fmaf(h[i], w.qw[i], w.qb[i]);
            c.store(a.normed, row, live, h);
        }
        if (a.stats && c.t == 0) {
            const u32x4 v = {__float_as_uint(st[0]), __float_as_uint(st[1]), __float_as_uint(st[2]), __float_as_uint(st[3])};
            __builtin_amdgcn_raw_buffer_store_b128(v, rows_rsrc(a.stats, row * 16, live ? 16 : 0), 0, 0, 0);
        }
    });
}

// Forward with one wave per row, where its registers hold the row: no barriers, the row sums stay inside the wave, and what a
// row costs besides its elements (addresses, reductions) is paid once per row instead of once per wave and row.  A lane holds
// NU units of 16 bytes, the wave's accesses are contiguous.  Every row is a wave of its own, dispatched in order, so that the
// rows in flight are neighbours in memory.  Against the row group kernel above: 65536 x 2304 bf16 norm alone 97 against
// 108 us (6.2 TB/s), 16384 x 2304 bf16 pair 51 against 58, fp32 102 against 110, 4096 x 2304 bf16 pair called in
// a row 12.3 against 13.3 (with inputs that no cache holds 18.9 against 17.4).
//   PLAIN: no bias and no gate per channel or element, which saves the registers of two rows.
template <int DT, int NU> struct WaveRow {
    static constexpr int E = DType<DT>::kVec;
    u32x4 r[NU];
    __device__ __forceinline__ void load(rsrc_t s, int lane, bool streaming) {
        if (streaming) {
#pragma unroll
            for (int u = 0; u < NU; ++u) r[u] = __builtin_amdgcn_raw_buffer_load_b128(s, (u * 64 + lane) * 16, 0, 2);
        } else {
#pragma unroll
            for (int u = 0; u < NU; ++u) r[u] = __builtin_amdgcn_raw_buffer_load_b128(s, (u * 64 + lane) * 16, 0, 0);
        }
    }
    __device__ __forceinline__ void unpack(int u, float (&v)[E]) const {
        if constexpr (DT == MTC_BF16) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __uint_as_float(r[u][i] << 16);
                v[2 * i + 1] = __uint_as_float(r[u][i] & 0xffff0000u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(r[u][i]);
        }
    }
    __device__ __forceinline__ void pack(int u, const float (&v)[E]) {
        if constexpr (DT == MTC_BF16) {
#pragma unroll
            for (int i = 0; i < 4; ++i) r[u][i] = pack2_bf16(v[2 * i], v[2 * i + 1]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) r[u][i] = __float_as_uint(v[i]);
        }
    }
    __device__ __forceinline__ void store(rsrc_t s, int lane, bool streaming) const {
        if (streaming) {
#pragma unroll
            for (int u = 0; u < NU; ++u) __builtin_amdgcn_raw_buffer_store_b128(r[u], s, (u * 64 + lane) * 16, 0, 2);
        } else {
#pragma unroll
            for (int u = 0; u < NU; ++u) __builtin_amdgcn_raw_buffer_store_b128(r[u], s, (u * 64 + lane) * 16, 0, 0);
        }
    }
};
// a lane's units added as a tree: with the 4 or 8 values of a unit one after another and 6 levels in the wave, a row sum has at
// most 18 roundings in sequence for any NU, where one chain over the lane's columns would have up to 78
template <int NU> __device__ __forceinline__ float units_total(float (&p)[NU]) {
#pragma unroll
    for (int s = 1; s < NU; s *= 2)
#pragma unroll
        for (int u = 0; u + s < NU; u += 2 * s) p[u] += p[u + s];
    return wave_total(p[0]);
}
// v becomes v - mean (layer); returns 1/std
template <int NU, int E>
__device__ __forceinline__ float wave_normalise(float (&v)[NU][E], int kind, float eps, float inv_A, int lane, int A, float& mu) {
    float p[NU];
    mu = 0.f;
    if (kind == MTC_NORM_LAYER) {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            p[u] = v[u][0];
#pragma unroll
            for (int i = 1; i < E; ++i) p[u] += v[u][i];
        }
        mu = units_total<NU>(p) * inv_A;
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const float m = (u * 64 + lane) * E < A ? mu : 0.f;
#pragma unroll
            for (int i = 0; i < E; ++i) v[u][i] -= m;
        }
    }
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        p[u] = v[u][0] * v[u][0];
#pragma unroll
        for (int i = 1; i < E; ++i) p[u] = fmaf(v[u][i], v[u][i], p[u]);
    }
    return 1.f / sqrtf(fmaf(units_total<NU>(p), inv_A, eps));
}

template <int DT, int NU, bool BRANCH, bool PRE, bool PLAIN>
__global__ __launch_bounds__(256, (BRANCH && NU <= 5 ? 4 : 1)) void block_norm_wave_kernel(NormArgs a) {
    constexpr int E = DType<DT>::kVec, ES = (int)sizeof(typename DType<DT>::T);
    typedef WaveRow<DT, NU> Row;
    const int lane = threadIdx.x & 63;
    const long long row = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)) + (long long)blockIdx.x * (blockDim.x >> 6);
    if (row >= a.rows) return;
    const int bytes = a.A * ES;
    const bool nt = a.streaming;
    auto rsrc = [&](const NormRow& o) { return rows_rsrc(o.p, row * o.ld * ES, bytes); };
    auto vec = [&](const void* p) { return rows_rsrc(p, 0, bytes); };
    Row r, y, g, w, b;
    r.load(rsrc(a.residual), lane, nt);
    if (BRANCH) y.load(rsrc(a.branch), lane, nt);
    float h[NU][E], t[E], st[4] = {0.f, 0.f, 0.f, 0.f};
    // h <- (h * rstd) * (offset + weight) + bias
    auto affine = [&](bool has_w, float off, bool has_b, float rstd) {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            if (has_w) {
                w.unpack(u, t);
#pragma unroll
                for (int i = 0; i < E; ++i) h[u][i] *= rstd * (off + t[i]);
            } else {
#pragma unroll
                for (int i = 0; i < E; ++i) h[u][i] *= rstd;
            }
            if (has_b) {
                b.unpack(u, t);
#pragma unroll
                for (int i = 0; i < E; ++i) h[u][i] += t[i];
            }
        }
    };
    if (BRANCH) {
        const bool post = a.post_kind != MTC_NORM_NONE, has_w = post && a.post_w, has_b = !PLAIN && post && a.post_b;
        const bool chan = !PLAIN && a.gate_kind == MTC_GATE_CHANNEL, full = !PLAIN && a.gate_kind == MTC_GATE_FULL;
        if (has_w) w.load(vec(a.post_w), lane, false);
        if (has_b) b.load(vec(a.post_b), lane, false);
        if (chan) g.load(vec(a.gate.p), lane, false);
        if (full) g.load(rsrc(a.gate), lane, nt);
        float scale = a.branch_scale;
        if (a.gate_kind == MTC_GATE_ROW || a.gate_kind == MTC_GATE_SCALAR)
            scale *= __uint_as_float(fetch_one<DT>(a.gate, row, true));
#pragma unroll
        for (int u = 0; u < NU; ++u) y.unpack(u, h[u]);
        if (post) {
            st[1] = wave_normalise<NU, E>(h, a.post_kind, a.post_eps, a.inv_A, lane, a.A, st[0]);
            affine(has_w, a.post_off, has_b, st[1]);
        }
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            if (chan || full) {
                g.unpack(u, t);
#pragma unroll
                for (int i = 0; i < E; ++i) h[u][i] *= t[i];
            }
            r.unpack(u, t);
#pragma unroll
            for (int i = 0; i < E; ++i) h[u][i] = fmaf(scale, h[u][i], a.res_scale * t[i]);
            r.pack(u, h[u]);
        }
        r.store(rsrc(a.hidden), lane, nt);
    } else {
#pragma unroll
        for (int u = 0; u < NU; ++u) r.unpack(u, h[u]);
    }
    if (PRE) {
        const bool has_w = a.pre_w, has_b = !PLAIN && a.pre_b;
        if (has_w) w.load(vec(a.pre_w), lane, false);
        if (has_b) b.load(vec(a.pre_b), lane, false);
        st[3] = wave_normalise<NU, E>(h, a.pre_kind, a.pre_eps, a.inv_A, lane, a.A, st[2]);
        affine(has_w, a.pre_off, has_b, st[3]);
#pragma unroll
        for (int u = 0; u < NU; ++u) y.pack(u, h[u]);
        y.store(rsrc(a.normed), lane, nt);
    }
    if (a.stats && lane == 0) {
        const u32x4 v = {__float_as_uint(st[0]), __float_as_uint(st[1]), __float_as_uint(st[2]), __float_as_uint(st[3])};
        *reinterpret_cast<u32x4*>(a.stats + row * 4) = v;
    }
}

// Gradient.  With g = d_normed, du = g (offset + w_pre):
//     D        = d_hidden + rstd (du - [layer] mean(du) - u mean(du u))          d_residual = residual_scale D
//     dv       = D gate pf                                                       (pf: branch scale x channel gate x post weight)
//     d_branch = rstd_p (dv - [layer] mean(dv) - u_p mean(dv u_p))               (post norm; else dv)
// and the column sums (over rows) X1 = gate D u_p, X2 = gate D, X3 = g u, X4 = g, from which block_norm_cols_kernel makes the
// gradients of the weights, biases and the channel gate.  Each workgroup leaves one partial per column, summed in a
// fixed order afterwards: no atomics, the same bits on every run.
// One workgroup per CU of up to 768 threads, several row groups in it where rows are short; its groups' sums meet in LDS.  168
// registers each hold the column sums, the weights and two rows' operands (fp32 pairs with a gate per element and biases spill 24).
// Rows above 6144 columns take up to 1024 threads with 128 registers: one row's operands, no prefetch, and pairs that keep
// all four sums spill 8 to 45 registers, but for aligned bf16 ones without a gate per element.  Bound by memory at large sizes:
// 16384 x 4608 bf16 pair with a channel gate 162 us with the column kernel (5.6 TB/s over its six operands), 16384 x 2304 84 us (5.4);
// by the operands' latency at small ones (1024 x 2304 15 us, 4096 x 2304 30) and without prefetch: 4096 x 8192 bf16 RMS pair 87 us
// (4.6 TB/s), layer norms 98, 4096 x 8191 in single elements 141.  A third row's operands in flight spill: 16384 x 1600 fp32
// 115 -> 167 us.
template <typename COLS, bool FULL> struct BwdRow {
    typename COLS::Raw branch, gate[FULL ? 1 : 0], d_hidden, residual, d_normed;
    uint32_t gr;
    u32x4 st;                            // the row's statistics
};

// SUMS: the column sums that are kept: 0 none, 1 X1 and X3, 2 all four (and the post norm's bias in z)
template <int DT, bool VEC, bool BRANCH, bool PRE, bool FULL, int SUMS, bool PREFETCH, int MAXT, bool STREAM>
__global__ __launch_bounds__(MAXT) void block_norm_bwd_kernel(NormArgs a) {
    typedef typename DType<DT>::T T_;
    __shared__ float sm[2 * 16 * 4];
    extern __shared__ float fold[];                      // (groups - 1) * T * 8 floats when SUMS > 0
    const int waves = a.T >> 6;
    const int group = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6) / waves);
    const Cols<DT, VEC, STREAM> c = {(int)threadIdx.x - group * a.T, a.T, a.A};
    int slot = 0;
    const bool gated = a.gate_kind == MTC_GATE_ROW || a.gate_kind == MTC_GATE_SCALAR;
    const long long base0 = (long long)blockIdx.x * a.groups, step = (long long)gridDim.x * a.groups;
    typedef BwdRow<Cols<DT, VEC, STREAM>, FULL> Row;
    auto fetch = [&](long long base, Row& q) {
        const bool live = base + group < a.rows;
        const long long row = live ? base + group : 0;
        q.st = __builtin_amdgcn_raw_buffer_load_b128(rows_rsrc(a.stats, row * 16, live && a.stats ? 16 : 0), 0, 0, 0);
        if (BRANCH) {
            c.fetch(a.branch, row, live, q.branch);
            c.fetch(a.d_hidden, row, live && a.d_hidden.p, q.d_hidden);
            if (FULL) c.fetch(a.gate, row, live, q.gate[0]);
            else q.gr = fetch_one<DT>(a.gate, row, live && gated);
        }
        if (PRE) {
            c.fetch(a.residual, row, live, q.residual);
            c.fetch(a.d_normed, row, live, q.d_normed);
        }
    };
    Row first;
    fetch(base0, first);
    NormWeights w;
    w.load(c, a, BRANCH, PRE);
    float x1[8], x2[8], x3[8], x4[8], gate_sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) x1[i] = x2[i] = x3[i] = x4[i] = 0.f;
    walk_rows<PREFETCH>(base0, step, a.rows, fetch, first, [&](long long base, const Row& q) {
        // Groups behind the last row read zeros everywhere, 1/std among them: they add zeros and store nothing.
        // An RMS norm's 1/std is folded into the factors of fused multiply-adds, and work that only a layer norm, a row gate, a
        // gate's gradient or a residual scale needs sits behind branches that the whole launch takes alike: the loop is
        // bound by the number of vector instructions once the loads are in flight in time.  A layer norm subtracts its mean
        // first, from the sum as the forward made it: x rstd - mu rstd would round at the size of mu for rows far from zero.
        const bool live = base + group < a.rows;
        const long long row = live ? base + group : 0;
        const float rstd_p = a.post_kind == MTC_NORM_NONE ? 1.f : __uint_as_float(q.st[1]);
        const float gr = FULL || !gated ? 1.f : __uint_as_float(q.gr);
        float D[8], up[8], z[8], g[8];
        if (BRANCH) {
            q.branch.unpack(up);
            if (a.post_kind == MTC_NORM_LAYER) {
                const float mu = __uint_as_float(q.st[0]);
#pragma unroll
                for (int i = 0; i < 8; ++i) up[i] = (up[i] - mu) * rstd_p;
            } else if (a.post_kind == MTC_NORM_RMS) {
#pragma unroll
                for (int i = 0; i < 8; ++i) up[i] *= rstd_p;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) z[i] = SUMS == 2 ? fmaf(up[i], w.pf[i], w.pb[i]) : up[i] * w.pf[i];
            if (FULL) q.gate[0].unpack(g);
            q.d_hidden.unpack(D);
        }
        if (PRE) {
            const float rstd = __uint_as_float(q.st[3]);
            float u[8], dn[8], s[2] = {0.f, 0.f};
            q.residual.unpack(u);
            q.d_normed.unpack(dn);
            if (a.pre_kind == MTC_NORM_LAYER) {
                const float mu = __uint_as_float(q.st[2]);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (BRANCH) u[i] = fmaf(FULL ? g[i] : gr, z[i], a.res_scale * u[i]);
                    u[i] = (u[i] - mu) * rstd;
                }
            } else {
                const float kr = BRANCH ? a.res_scale * rstd : rstd, kz = gr * rstd;
#pragma unroll
                for (int i = 0; i < 8; ++i) u[i] = BRANCH ? fmaf(kr, u[i], (FULL ? g[i] * rstd : kz) * z[i]) : kr * u[i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (SUMS >= 1) x3[i] = fmaf(dn[i], u[i], x3[i]);
                if (SUMS >= 2) x4[i] += dn[i];
                dn[i] *= w.qw[i];
                s[0] = fmaf(dn[i], u[i], s[0]);
            }
            if (a.pre_kind == MTC_NORM_LAYER) {
#pragma unroll
                for (int i = 0; i < 8; ++i) s[1] += dn[i];
                group_sum(s, sm, slot, group, waves);
                const float m1 = -s[1] * a.inv_A;
#pragma unroll
                for (int i = 0; i < 8; ++i) dn[i] += m1;
            } else {
                float s1[1] = {s[0]};
                group_sum(s1, sm, slot, group, waves);
                s[0] = s1[0];
            }
            const float m2 = -s[0] * a.inv_A * rstd;
#pragma unroll
            for (int i = 0; i < 8; ++i) D[i] = fmaf(m2, u[i], BRANCH ? fmaf(rstd, dn[i], D[i]) : rstd * dn[i]);
        }
        if (BRANCH && a.res_scale != 1.f) {
            float o[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = a.res_scale * D[i];
            c.store(a.d_residual, row, live && a.d_residual.p, o);
        } else {
            c.store(a.d_residual, row, live && a.d_residual.p, D);
        }
        if (BRANCH) {
            float s[3] = {0.f, 0.f, 0.f};
            const bool row_sum = (a.gate_kind == MTC_GATE_ROW && a.d_gate.p) || a.want_scalar;
            if (FULL || row_sum) {                       // d gate, before its reduction
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    z[i] *= D[i];
                    s[2] += z[i];
                }
            }
            if (FULL) c.store(a.d_gate, row, live && a.d_gate.p, z);
            if (FULL || gated) {
#pragma unroll
                for (int i = 0; i < 8; ++i) D[i] *= FULL ? g[i] : gr;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (SUMS >= 1) x1[i] = fmaf(D[i], up[i], x1[i]);
                if (SUMS >= 2) x2[i] += D[i];
                D[i] *= w.pf[i];
            }
            if (a.post_kind != MTC_NORM_NONE) {
#pragma unroll
                for (int i = 0; i < 8; ++i) s[1] = fmaf(D[i], up[i], s[1]);
            }
            if (row_sum || a.post_kind == MTC_NORM_LAYER) {
#pragma unroll
                for (int i = 0; i < 8; ++i) s[0] += D[i];
                group_sum(s, sm, slot, group, waves);
                if (a.gate_kind == MTC_GATE_ROW && a.d_gate.p && live && c.t == 0)
                    DType<DT>::st(reinterpret_cast<T_*>(a.d_gate.p) + row, s[2]);
                gate_sum += s[2];
            } else if (a.post_kind == MTC_NORM_RMS) {
                float s1[1] = {s[1]};
                group_sum(s1, sm, slot, group, waves);
                s[1] = s1[0];
            }
            if (a.post_kind != MTC_NORM_NONE) {
                const float m1 = a.post_kind == MTC_NORM_LAYER ? -s[0] * a.inv_A * rstd_p : 0.f, m2 = -s[1] * a.inv_A * rstd_p;
#pragma unroll
                for (int i = 0; i < 8; ++i) D[i] = fmaf(m2, up[i], fmaf(rstd_p, D[i], m1));
            }
            c.store(a.d_branch, row, live && a.d_branch.p, D);
        }
    });
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
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (c.in(i)) out[(size_t)which * a.pitch + c.col(i)] = x[i];
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

// the last sums over the workgroups' partials: 64 columns per workgroup, its 16 waves share the partials.  Bound by latency
// (width 4608: 13 MB of partials in 5 us)
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

constexpr int NORM_BWD_T = 768;                    // threads of a backward workgroup, if a row needs no more: 168 registers each
constexpr long long WAVE_MAX_ROWS = 1ll << 25;             // one wave each: a launch has at most 2^32 threads
constexpr long long NORM_STREAM_BYTES = 256ll << 20;       // the Infinity Cache

// workgroups for `want` row sets: at most per_cu on each CU, and every one the same number of rounds
static unsigned norm_grid(long long want, int per_cu) {
    const long long most = (long long)NORM_CUS * (per_cu < 1 ? 1 : per_cu);
    if (want <= most) return (unsigned)want;
    const long long rounds = (want + most - 1) / most;
    return (unsigned)((want + rounds - 1) / rounds);
}

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
    return (d->A & (16 / norm_elem(d->dtype) - 1)) == 0 && row_vec(a.residual.p, a.residual.ld, d->rows, d->dtype) &&
           row_vec(a.branch.p, a.branch.ld, d->rows, d->dtype) &&
           ((a.gate_kind != MTC_GATE_CHANNEL && a.gate_kind != MTC_GATE_FULL) ||
            row_vec(a.gate.p, a.gate_kind == MTC_GATE_FULL ? a.gate.ld : 0, d->rows, d->dtype)) &&
           row_vec(a.post_w, 0, 1, d->dtype) && row_vec(a.post_b, 0, 1, d->dtype) && row_vec(a.pre_w, 0, 1, d->dtype) &&
           row_vec(a.pre_b, 0, 1, d->dtype);
}

template <int DT, bool VEC, bool STREAM> static void launch_norm_fwd(const NormArgs& a, bool branch, unsigned grid, hipStream_t s) {
    const dim3 b(a.T * a.groups), g(grid);
    const bool pre = a.pre_kind != MTC_NORM_NONE, full = a.gate_kind == MTC_GATE_FULL;
    if (!branch) hipLaunchKernelGGL((block_norm_fwd_kernel<DT, VEC, false, true, false, STREAM>), g, b, 0, s, a);
    else if (pre && full) hipLaunchKernelGGL((block_norm_fwd_kernel<DT, VEC, true, true, true, STREAM>), g, b, 0, s, a);
    else if (pre) hipLaunchKernelGGL((block_norm_fwd_kernel<DT, VEC, true, true, false, STREAM>), g, b, 0, s, a);
    else if (full) hipLaunchKernelGGL((block_norm_fwd_kernel<DT, VEC, true, false, true, STREAM>), g, b, 0, s, a);
    else hipLaunchKernelGGL((block_norm_fwd_kernel<DT, VEC, true, false, false, STREAM>), g, b, 0, s, a);
}

// What a wave can hold: 9 units a lane for a norm alone; with a branch 40 floats of a row, 36 where biases or a gate per
// channel or element need rows of their own.  Row groups against one wave per row, us:
//   beyond: bf16 pair 3584 wide 23.6 / 27.3 (4096 rows), 77.6 / 78.7 (16384); 4608 wide 29.9 / 33.7, 97.0 / 100.2; bf16 layer norms with a
//           channel gate 2304 wide 19.5 / 26.4, 65.0 / 77.6
//   within: bf16 pair 2304 wide 57.6 / 51.0 (16384 rows); fp32 1600 wide 76.9 / 71.1, 2304 wide 110 / 102, with layer norms 116 / 101.  Only
//           around 4096 rows, read from memory, are row groups ahead by up to 2.5 us (17.4 / 18.9, fp32 layer norms 32.7 / 35.2)
template <int DT, bool BRANCH, bool PLAIN> constexpr int wave_units() {
    return !BRANCH ? 9 : std::min(9, (PLAIN ? 40 : 36) / DType<DT>::kVec);
}

template <int DT, int NU, bool PLAIN> static bool launch_norm_wave(const NormArgs& a, bool branch, hipStream_t s) {
    const int per = a.rows < 4 * NORM_CUS ? 1 : 4;
    const dim3 g((unsigned)((a.rows + per - 1) / per)), b(64 * per);
    if (!branch) {
        hipLaunchKernelGGL((block_norm_wave_kernel<DT, NU, false, true, PLAIN>), g, b, 0, s, a);
        return true;
    }
    if constexpr (NU <= wave_units<DT, true, PLAIN>()) {
        if (a.pre_kind != MTC_NORM_NONE) hipLaunchKernelGGL((block_norm_wave_kernel<DT, NU, true, true, PLAIN>), g, b, 0, s, a);
        else hipLaunchKernelGGL((block_norm_wave_kernel<DT, NU, true, false, PLAIN>), g, b, 0, s, a);
        return true;
    }
    return false;
}

template <int DT, bool PLAIN> static bool launch_norm_wave_units(const NormArgs& a, bool branch, hipStream_t s) {
    switch ((a.A * norm_elem(DT) + 1023) / 1024) {
        case 1: return launch_norm_wave<DT, 1, PLAIN>(a, branch, s);
        case 2: return launch_norm_wave<DT, 2, PLAIN>(a, branch, s);
        case 3: return launch_norm_wave<DT, 3, PLAIN>(a, branch, s);
        case 4: case 5: return launch_norm_wave<DT, 5, PLAIN>(a, branch, s);
        case 6: case 7: return launch_norm_wave<DT, 7, PLAIN>(a, branch, s);
        case 8: case 9: return launch_norm_wave<DT, 9, PLAIN>(a, branch, s);
        default: return false;
    }
}

template <int DT> static void launch_norm_fwd_dt(const NormArgs& a, bool branch, bool vec, unsigned grid, hipStream_t s) {
    const bool plain = !a.post_b && !a.pre_b && a.gate_kind != MTC_GATE_CHANNEL && a.gate_kind != MTC_GATE_FULL;
    if (vec && a.rows <= WAVE_MAX_ROWS && (plain ? launch_norm_wave_units<DT, true>(a, branch, s) : launch_norm_wave_units<DT, false>(a, branch, s)))
        return;
    if (!vec) launch_norm_fwd<DT, false, false>(a, branch, grid, s);
    else if (a.streaming) launch_norm_fwd<DT, true, true>(a, branch, grid, s);
    else launch_norm_fwd<DT, true, false>(a, branch, grid, s);
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
    MTC_REQUIRE(!stats || ((uintptr_t)stats & 15) == 0, "%s: stats must be 16-byte aligned", who);
    a.hidden = {hidden, d->ld_hidden};
    a.normed = {normed, d->ld_normed};
    a.post_w = post_w; a.post_b = post_b; a.pre_w = pre_w; a.pre_b = pre_b;
    a.stats = stats;
    const bool vec = norm_inputs_vec(d, a) && row_vec(hidden, d->ld_hidden, d->rows, d->dtype) &&
                     row_vec(normed, d->ld_normed, d->rows, d->dtype);
    a.groups = a.T >= 256 ? 1 : 256 / a.T;
    // operands read and written once; beyond the Infinity Cache non-temporal accesses and, for two RMS norms (whose rows wait
    // least), few waves that keep to few DRAM pages are faster: 16384 x 4608 bf16 pair 97 against 118 us.  Within the cache the
    // opposite holds: 4096 x 2304 pair 14.8 against 17.0 us, and what follows finds plain stores in the cache (four such
    // calls in a row 60 against 65 us).  12 / 20 / 28 waves per CU, us:
    //   beyond, RMS:   16384 x 4608 bf16 97 / 113 / 108, 16384 x 4096 fp32 179 / 181 / 190, 65536 x 1001 bf16 111 / 117 / 120
    //   beyond, layer: 16384 x 4608 bf16 134 / 116 / 116, 65536 x 1001 bf16 124 / 122 / 124, 32768 x 2304 bf16 127 / 130 / 129; 16384 x 4096 fp32
    //                  183 / 186 / 197, where 28 is 7 % behind
    //   within:        4096 x 4608 bf16 30.0 / 30.1 / 31.9, 1024 x 4608 10.9 / 10.5 / 10.5, 8192 x 1001 19.5 / 18.6 / 20.1
    // Above 6144 columns a row takes 13 waves or more, and all three mean one workgroup per CU.
    const int passes = (branch ? 2 : 1) + (d->gate_kind == MTC_GATE_FULL) + (hidden != nullptr) + (normed != nullptr);
    a.streaming = d->rows * d->A * norm_elem(d->dtype) * passes > NORM_STREAM_BYTES;
    const bool layer = d->post_kind == MTC_NORM_LAYER || d->pre_kind == MTC_NORM_LAYER;
    const int waves = !a.streaming ? 20 : branch && !layer ? 12 : 28;
    const unsigned grid = norm_grid((d->rows + a.groups - 1) / a.groups, waves / (a.T * a.groups / 64));
    hipStream_t s = as_stream(stream);
    if (d->dtype == MTC_BF16) launch_norm_fwd_dt<MTC_BF16>(a, branch, vec, grid, s);
    else launch_norm_fwd_dt<MTC_F32>(a, branch, vec, grid, s);
    return check_launch(who);
}

// backward launch shape: one workgroup per CU of up to 1024 threads, fewer row groups when there are few rows
static void norm_bwd_shape(const mtc_block_norm_desc* d, int& groups, unsigned& grid) {
    const int T = norm_threads(d->A), most = T > NORM_BWD_T ? 1 : NORM_BWD_T / T;
    const long long per_cu = (d->rows + NORM_CUS - 1) / NORM_CUS;
    groups = (int)(per_cu < most ? per_cu : most);
    grid = norm_grid((d->rows + groups - 1) / groups, 1);
}

extern "C" size_t mtc_block_norm_bwd_workspace_bytes(const mtc_block_norm_desc* d) {
    if (norm_check(d, "mtc_block_norm_bwd_workspace_bytes")) return 0;
    if (d->rows == 0) return 0;
    int groups;
    unsigned grid;
    norm_bwd_shape(d, groups, grid);
    return (size_t)grid * (4 * ((d->A + 7) / 8 * 8) + 8) * sizeof(float);
}

template <int DT, bool VEC, bool BRANCH, bool PRE, bool FULL, bool PREFETCH, int MAXT, bool STREAM>
static void launch_norm_bwd_sums(const NormArgs& a, int sums, unsigned grid, hipStream_t s) {
    const dim3 b(a.T * a.groups), g(grid);
    const size_t lds = sums ? (size_t)(a.groups - 1) * a.T * 8 * sizeof(float) : 0;
    if (sums == 0) hipLaunchKernelGGL((block_norm_bwd_kernel<DT, VEC, BRANCH, PRE, FULL, 0, PREFETCH, MAXT, STREAM>), g, b, lds, s, a);
    else if (VEC && sums == 1)
        hipLaunchKernelGGL((block_norm_bwd_kernel<DT, VEC, BRANCH, PRE, FULL, VEC ? 1 : 2, PREFETCH, MAXT, STREAM>), g, b, lds, s, a);
    else hipLaunchKernelGGL((block_norm_bwd_kernel<DT, VEC, BRANCH, PRE, FULL, 2, PREFETCH, MAXT, STREAM>), g, b, lds, s, a);
}

template <int DT, bool VEC, bool BRANCH, bool PRE, bool FULL>
static void launch_norm_bwd(const NormArgs& a, int sums, bool streaming, unsigned grid, hipStream_t s) {
    if (a.T * a.groups > NORM_BWD_T) launch_norm_bwd_sums<DT, VEC, BRANCH, PRE, FULL, false, 1024, false>(a, sums, grid, s);
    // gates per element have no streaming instance: beyond the cache that costs 8 % (16384 x 2304 fp32 pair 233 against 215 us, bf16
    // 118 against 108), within it nothing
    else if (VEC && !FULL && streaming) launch_norm_bwd_sums<DT, VEC, BRANCH, PRE, FULL, VEC, NORM_BWD_T, VEC && !FULL>(a, sums, grid, s);
    else launch_norm_bwd_sums<DT, VEC, BRANCH, PRE, FULL, VEC, NORM_BWD_T, false>(a, sums, grid, s);
}

template <int DT, bool VEC>
static void launch_norm_bwd_mode(const NormArgs& a, bool branch, int sums, bool streaming, unsigned grid, hipStream_t s) {
    const bool pre = a.pre_kind != MTC_NORM_NONE, full = a.gate_kind == MTC_GATE_FULL;
    if (!branch) launch_norm_bwd<DT, VEC, false, true, false>(a, sums, streaming, grid, s);
    else if (pre && full) launch_norm_bwd<DT, VEC, true, true, true>(a, sums, streaming, grid, s);
    else if (pre) launch_norm_bwd<DT, VEC, true, true, false>(a, sums, streaming, grid, s);
    else if (full) launch_norm_bwd<DT, VEC, true, false, true>(a, sums, streaming, grid, s);
    else launch_norm_bwd<DT, VEC, true, false, false>(a, sums, streaming, grid, s);
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
    MTC_REQUIRE(!stats || ((uintptr_t)stats & 15) == 0, "%s: stats must be 16-byte aligned", who);
    MTC_REQUIRE(ld_d_hidden >= 0 && ld_d_normed >= 0, "%s: negative row stride", who);
    a.post_w = post_w; a.post_b = post_b; a.pre_w = pre_w; a.pre_b = pre_b;
    a.stats = const_cast<float*>(stats);
    a.d_hidden = {const_cast<void*>(d_hidden), ld_d_hidden};
    a.d_normed = {const_cast<void*>(d_normed), ld_d_normed};
    a.d_residual = {d_residual, d->A};
    a.d_branch = {d_branch, d->A};
    a.d_gate = {d_gate, d->A};
    const bool chan = d->gate_kind == MTC_GATE_CHANNEL && d_gate;
    const bool chan_bias = chan && d->post_kind != MTC_NORM_NONE && post_b;
    a.want_x1 = d_post_w || chan;
    a.want_x2 = d_post_b || chan_bias;
    a.want_x3 = d_pre_w != nullptr;
    a.want_x4 = d_pre_b != nullptr;
    a.want_scalar = d->gate_kind == MTC_GATE_SCALAR && d_gate;
    const bool any_sum = a.want_x1 || a.want_x2 || a.want_x3 || a.want_x4 || a.want_scalar;
    // 2: also whenever the branch's norm has a bias, which the smaller forms leave out of the recomputed branch
    const int sums = a.want_x2 || a.want_x4 || (d->post_kind != MTC_NORM_NONE && post_b) ? 2 : any_sum ? 1 : 0;
    a.pitch = (d->A + 7) / 8 * 8;
    unsigned grid;
    norm_bwd_shape(d, a.groups, grid);
    if (any_sum) {
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
    // non-temporal beyond the Infinity Cache: 16384 x 4608 bf16 pair 158 against 174 us; 1024 x 768 fp32, within it: 12.4
    // against 10.8 us
    const int passes = (branch ? 1 : 0) + (d_hidden != nullptr) + (d->pre_kind != MTC_NORM_NONE ? 2 : 0) + (d_residual != nullptr) +
                       (d_branch != nullptr);
    const bool streaming = d->rows * A * norm_elem(d->dtype) * passes > NORM_STREAM_BYTES;
    if (d->dtype == MTC_BF16)
        vec ? launch_norm_bwd_mode<MTC_BF16, true>(a, branch, sums, streaming, grid, s) : launch_norm_bwd_mode<MTC_BF16, false>(a, branch, sums, streaming, grid, s);
    else
        vec ? launch_norm_bwd_mode<MTC_F32, true>(a, branch, sums, streaming, grid, s) : launch_norm_bwd_mode<MTC_F32, false>(a, branch, sums, streaming, grid, s);
    if (check_launch(who)) return -2;
    if (any_sum) {
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
