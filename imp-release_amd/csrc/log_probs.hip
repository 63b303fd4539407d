// Log probabilities of given matches, with entropy and the best alternatives, and their gradient (C-ABI imp_log_probs_forward / _backward; gfx950).
// Row by row over logits x [rows][cols] (fp32 / fp16 / bf16), with an optional dustbin: one more column of the same value in every row (the matcher's bin_score):
//   m = max x, l = log sum exp(x - m)     logp = (x_t - m) - l     H = l + sum p (m - x)     the `top` largest columns, ties to the lower index
//   dx_j = g (delta_jt - p_j) - h p_j (logp_j + H)                 g, h: the gradients of logp and H
// The sum leaves the largest element out, l = log1p(s): the log probability of a sure match is near 0, and 1 + s would round it away (and with it H and 1 - p,
// which is -expm1(logp)).  Columns of -inf are masked: no probability, never an alternative; a row of nothing else has logp = -inf, H = 0 and no gradient.
//
// Forward: one pass over the row.  A thread keeps (m, s, U = sum e (m - x)) of its elements; two such states join as
//   m = max, s = s_a + (s_b + 1) f, U = U_a + f (U_b + d (s_b + 1)), f = exp(-d), d = m_a - m_b >= 0            (the smaller maximum becomes an ordinary element)
// lanes, waves and - when there are few rows - shares of a row are joined in a fixed order.  Bound by reading the logits.
#include "../../include/imp_hip.h"
#include "imp_kernels.h"

int imp_fail(int code, const char* msg);   // context.hip: sets imp_last_error()

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int TOP_MAX = 16;

struct LogpOp {
    const void* x;
    const int64_t* target;
    const float* bin;
    float *logp, *entropy, *stats, *top_logp;
    int64_t* top_id;
    const float *dlogp, *dentropy;
    void* dx;
    float* dbin;
    int64_t rows, ld;
    int cols, top, shares;
    float* part;                         // per share: m, s, U
    float* part_v;
    int* part_i;
    double* part_bin;
};

__device__ __forceinline__ float exp_neg(float d) { return __builtin_amdgcn_exp2f(d * LOG2E); }

struct State { float m, s, u; };
__device__ __forceinline__ State empty_state() { return {-INFINITY, 0.f, 0.f}; }
// the order of the operands does not change which elements are summed; equal maxima count a's as the one left out
__device__ __forceinline__ State join(State a, State b) {
    if (b.m > a.m) { const State t = a; a = b; b = t; }
    if (b.m == -INFINITY) return a;
    const float d = fminf(a.m - b.m, 1e30f), f = exp_neg(-d), n = b.s + 1.f;       // two of the type's extremes are further apart than it reaches
    return {a.m, a.s + n * f, a.u + f * (b.u + d * n)};
}
__device__ __forceinline__ State shfl_state(State a, int o) { return {__shfl_xor(a.m, o), __shfl_xor(a.s, o), __shfl_xor(a.u, o)}; }

// the K best (value, index) of a thread, best first; index INT_MAX marks an empty place
template <int K> struct Best {
    float v[K ? K : 1];
    int i[K ? K : 1];
    __device__ void clear() {
#pragma unroll
        for (int k = 0; k < K; ++k) { v[k] = -INFINITY; i[k] = 0x7fffffff; }
    }
    // elements come in rising index order per thread: a tie goes behind
    __device__ void take(float x, int at) {
        if (K == 0 || !(x > v[K ? K - 1 : 0])) return;
#pragma unroll
        for (int k = K - 1; k >= 0; --k) {
            const bool up = k > 0 && x > v[k > 0 ? k - 1 : 0];
            const float nv = up ? v[k > 0 ? k - 1 : 0] : x;
            const int ni = up ? i[k > 0 ? k - 1 : 0] : at;
            if (x > v[k]) { v[k] = nv; i[k] = ni; }
        }
    }
    __device__ void pop() {
#pragma unroll
        for (int k = 0; k + 1 < K; ++k) { v[k] = v[k + 1]; i[k] = i[k + 1]; }
        if (K) { v[K - 1] = -INFINITY; i[K - 1] = 0x7fffffff; }
    }
};
__device__ __forceinline__ bool better(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

template <typename T> __device__ __forceinline__ float to_f(T v) { return (float)v; }

// calls f(index, value) for this thread's elements of [c0, c1) in rising order: single elements up to the first 16-byte boundary, then vectors, then the rest
template <typename T, typename F, typename G>
__device__ __forceinline__ void walk(const T* x, int c0, int c1, int tid, int threads, F one, G vec) {
    constexpr int V = 16 / sizeof(T);
    const int head0 = (int)((16 - ((uintptr_t)(x + c0) & 15)) & 15) / (int)sizeof(T);
    const int head = head0 < c1 - c0 ? head0 : c1 - c0;
    const int body = (c1 - c0 - head) / V;
    if (tid < head) one(c0 + tid, to_f(x[c0 + tid]));
    for (int i = tid; i < body; i += threads) vec(c0 + head + i * V);
    const int tail = c0 + head + body * V + tid;
    if (tail < c1) one(tail, to_f(x[tail]));
}
template <typename T> struct alignas(16) Vec { T v[16 / sizeof(T)]; };

// W waves per row (W = 1: four rows per workgroup); one row or share of a row per group
template <typename T, int K, int W>
__global__ __launch_bounds__(256) void logp_forward_kernel(LogpOp p) {
    constexpr int V = 16 / sizeof(T), THREADS = 64 * W, GROUPS = 4 / W;
    __shared__ State sm_state[4];
    __shared__ float sm_v[4][K ? K : 1];
    __shared__ int sm_i[4][K ? K : 1];
    const int tid = threadIdx.x % THREADS, group = threadIdx.x / THREADS, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = (int64_t)blockIdx.x * GROUPS + group;
    if (W == 1 && row >= p.rows) return;
    const int share = blockIdx.y;
    const int c0 = (int)((int64_t)p.cols * share / p.shares), c1 = (int)((int64_t)p.cols * (share + 1) / p.shares);
    const T* x = (const T*)p.x + row * p.ld;
    State st = empty_state();
    Best<K> best;
    best.clear();
    bool bad = false;
    auto one = [&](int at, float v) {
        if (v != v) bad = true;
        else if (v != -INFINITY) st = join(st, {v, 0.f, 0.f});
        if (K) best.take(v, at);
    };
    walk<T>(x, c0, c1, tid, THREADS, one, [&](int at) {
        const Vec<T> v = *(const Vec<T>*)(x + at);
        float f[V], mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < V; ++i) { f[i] = to_f(v.v[i]); mx = fmaxf(mx, f[i]); }
        if (mx > st.m) {                 // a new maximum of this thread: it leaves the sum, the old one enters it
            State nw = {mx, 0.f, 0.f};
            bool out = false;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const bool self = f[i] == mx && !out;
                out |= self;
                const float d = f[i] - mx, e = self || f[i] == -INFINITY ? 0.f : exp_neg(d);
                nw.s += e;
                nw.u -= e == 0.f ? 0.f : e * d;
                bad |= f[i] != f[i];
            }
            st = join(nw, st);
        } else if (st.m != -INFINITY) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = f[i] - st.m, e = exp_neg(d);
                st.s += e;
                st.u -= e == 0.f ? 0.f : e * d;         // NaN logits pass through e
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) bad |= f[i] != f[i];
        }
        if (K) {
#pragma unroll
            for (int i = 0; i < V; ++i) best.take(f[i], at + i);
        }
    });
    if (p.bin && share == p.shares - 1 && tid == 0) one(p.cols, *p.bin);
    if (bad) { st.s = NAN; st.u = NAN; }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const State b = shfl_state(st, o);
        st = (lane & o) ? join(b, st) : join(st, b);
    }
    // NaN states survive a join only through s: a lane that saw nothing but NaN has m = -inf, so the flag is carried beside it
    const bool any_bad = __ballot(bad) != 0;
    float bv[K ? K : 1];
    int bi[K ? K : 1];
    if (K) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            float v = best.v[0];
            int i = best.i[0];
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const float w = __shfl_xor(v, o);
                const int j = __shfl_xor(i, o);
                if (better(w, j, v, i)) { v = w; i = j; }
            }
            bv[k] = v;
            bi[k] = i;
            if (best.i[0] == i) best.pop();
        }
    }
    if (any_bad || st.m == INFINITY) { st.s = NAN; st.u = NAN; if (st.m == -INFINITY) st.m = 0.f; }
    if (W > 1) {
        if (lane == 0) {
            sm_state[wave] = st;
#pragma unroll
            for (int k = 0; k < K; ++k) { sm_v[wave][k] = bv[k]; sm_i[wave][k] = bi[k]; }
        }
        __syncthreads();
        if (threadIdx.x != 0) return;
        st = sm_state[0];
        for (int w = 1; w < W; ++w) st = join(st, sm_state[w]);
        if (K) {
            int at[4] = {0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < K; ++k) {
                int from = 0;
                float v = -INFINITY;
                int i = 0x7fffffff;
                for (int w = 0; w < W; ++w)
                    if (at[w] < K && better(sm_v[w][at[w]], sm_i[w][at[w]], v, i)) { v = sm_v[w][at[w]]; i = sm_i[w][at[w]]; from = w; }
                for (int w = 0; w < W; ++w) at[w] += w == from;
                bv[k] = v;
                bi[k] = i;
            }
        }
    } else if (lane != 0) return;
    if (p.shares > 1) {
        const int64_t at = row * p.shares + share;
        p.part[3 * at] = st.m;
        p.part[3 * at + 1] = st.s;
        p.part[3 * at + 2] = st.u;
#pragma unroll
        for (int k = 0; k < K; ++k) { p.part_v[at * K + k] = bv[k]; p.part_i[at * K + k] = bi[k]; }
        return;
    }
    const float l = log1pf(st.s);
    const bool none = st.m == -INFINITY;
    p.stats[2 * row] = st.m;
    p.stats[2 * row + 1] = l;
    p.entropy[row] = none ? 0.f : l + st.u / (1.f + st.s);
    const int64_t t = p.target[row];
    float lp = 0.f;
    if (t >= 0 && t < p.cols) lp = none ? -INFINITY : (to_f(x[t]) - st.m) - l;
    else if (p.bin && (t == -1 || t == p.cols)) lp = none ? -INFINITY : (*p.bin - st.m) - l;
    else if (t != -1 && t != -2) lp = NAN;
    p.logp[row] = lp;
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (k < p.top) {
            const bool has = bv[k] != -INFINITY;
            p.top_logp[row * p.top + k] = has ? (bv[k] - st.m) - l : -INFINITY;
            p.top_id[row * p.top + k] = has ? bi[k] : -1;
        }
}

// joins the shares of a row (one wave per row)
template <typename T, int K>
__global__ __launch_bounds__(256) void logp_join_kernel(LogpOp p) {
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= p.rows) return;
    State st = empty_state();
    Best<K> best;
    best.clear();
    if (lane < p.shares) {
        const int64_t at = row * p.shares + lane;
        st = {p.part[3 * at], p.part[3 * at + 1], p.part[3 * at + 2]};
#pragma unroll
        for (int k = 0; k < K; ++k) { best.v[k] = p.part_v[at * K + k]; best.i[k] = p.part_i[at * K + k]; }
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const State b = shfl_state(st, o);
        st = (lane & o) ? join(b, st) : join(st, b);
    }
    const float l = log1pf(st.s);
    const bool none = st.m == -INFINITY;
    for (int k = 0; k < p.top; ++k) {
        float v = K ? best.v[0] : -INFINITY;
        int i = K ? best.i[0] : 0x7fffffff;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const float w = __shfl_xor(v, o);
            const int j = __shfl_xor(i, o);
            if (better(w, j, v, i)) { v = w; i = j; }
        }
        if (K && best.i[0] == i) best.pop();
        if (lane == 0) {
            const bool has = v != -INFINITY;
            p.top_logp[row * p.top + k] = has ? (v - st.m) - l : -INFINITY;
            p.top_id[row * p.top + k] = has ? i : -1;
        }
    }
    if (lane) return;
    p.stats[2 * row] = st.m;
    p.stats[2 * row + 1] = l;
    p.entropy[row] = none ? 0.f : l + st.u / (1.f + st.s);
    const int64_t t = p.target[row];
    const T* x = (const T*)p.x + row * p.ld;
    float lp = 0.f;
    if (t >= 0 && t < p.cols) lp = none ? -INFINITY : (to_f(x[t]) - st.m) - l;
    else if (p.bin && (t == -1 || t == p.cols)) lp = none ? -INFINITY : (*p.bin - st.m) - l;
    else if (t != -1 && t != -2) lp = NAN;
    p.logp[row] = lp;
}

// dx of one row, or of a share of it
template <typename T, int W>
__global__ __launch_bounds__(256) void logp_backward_kernel(LogpOp p) {
    constexpr int V = 16 / sizeof(T), THREADS = 64 * W, GROUPS = 4 / W;
    const int tid = threadIdx.x % THREADS, group = threadIdx.x / THREADS;
    const int64_t row = (int64_t)blockIdx.x * GROUPS + group;
    if (row >= p.rows) return;
    const int share = blockIdx.y;
    const T* x = (const T*)p.x + row * p.ld;
    T* dx = p.dx ? (T*)p.dx + row * p.cols : nullptr;
    int c0 = (int)((int64_t)p.cols * share / p.shares), c1 = (int)((int64_t)p.cols * (share + 1) / p.shares);
    const float m = p.stats[2 * row], l = p.stats[2 * row + 1], H = p.entropy[row];
    const bool none = m == -INFINITY;
    int64_t t = p.target[row];
    if (p.bin && t == -1) t = p.cols;
    const bool has = t >= 0 && t < p.cols + (p.bin ? 1 : 0);
    float g = p.dlogp && (has || (t != -1 && t != -2)) ? p.dlogp[row] : 0.f;
    if (!has && t != -1 && t != -2) g = NAN;
    const float h = p.dentropy ? p.dentropy[row] : 0.f;
    const int ti = has ? (int)t : -1;
    auto grad = [&](int at, float v) {
        if (none) return 0.f;
        const float lp = (v - m) - l, pr = exp_neg(lp);
        const float ent = pr == 0.f ? 0.f : h * (pr * (lp + H));
        return (at == ti ? -g * expm1f(lp) : -g * pr) - ent;
    };
    if (dx) {
        if ((((uintptr_t)x ^ (uintptr_t)dx) & 15) == 0) {
            walk<T>(x, c0, c1, tid, THREADS, [&](int at, float v) { dx[at] = (T)grad(at, v); },
                    [&](int at) {
                        const Vec<T> v = *(const Vec<T>*)(x + at);
                        Vec<T> o;
                        if (ti >= at && ti < at + V) {
#pragma unroll
                            for (int i = 0; i < V; ++i) o.v[i] = (T)grad(at + i, to_f(v.v[i]));
                        } else {
#pragma unroll
                            for (int i = 0; i < V; ++i) o.v[i] = (T)grad(-2, to_f(v.v[i]));
                        }
                        *(Vec<T>*)(dx + at) = o;
                    });
        } else {
            for (int i = c0 + tid; i < c1; i += THREADS) dx[i] = (T)grad(i, to_f(x[i]));
        }
    }
    if (p.bin && p.part_bin && share == 0 && tid == 0) p.part_bin[row] = (double)grad(p.cols, *p.bin);
}

// dbin = sum over the rows, in a fixed order
__global__ __launch_bounds__(1024) void logp_bin_kernel(const double* part, int64_t rows, float* out) {
    __shared__ double sm[1024];
    double a = 0;
    for (int64_t i = threadIdx.x; i < rows; i += 1024) a += part[i];
    sm[threadIdx.x] = a;
    for (int o = 512; o > 0; o >>= 1) {
        __syncthreads();
        if (threadIdx.x < o) sm[threadIdx.x] += sm[threadIdx.x + o];
    }
    if (threadIdx.x == 0) *out = (float)sm[0];
}

// ------------------------------------------------------------------------------------------------------------------------- host
// shares of a row: enough workgroups for four per CU, each with at least 4096 columns; at most 64 (a lane each in the join)
int shares_of(int64_t rows, int cols) {
    const int64_t want = (1024 + rows - 1) / rows, most = cols / 4096;
    const int64_t s = want < most ? want : most;
    return s < 1 ? 1 : (s > 64 ? 64 : (int)s);
}
int padded_top(int top) { return top == 0 ? 0 : top <= 1 ? 1 : top <= 4 ? 4 : top <= 8 ? 8 : TOP_MAX; }
// a wave per row where rows are short or there are plenty of them; four waves otherwise
bool wave_rows(int64_t rows, int cols) { return cols <= 512 || (cols <= 4096 && rows >= 4096); }

const char* bad(int dtype, int64_t rows, int cols, int64_t ld, const void* x, bool bin) {
    if (dtype != IMP_DTYPE_F32 && dtype != IMP_DTYPE_F16 && dtype != IMP_DTYPE_BF16) return "unknown dtype";
    if (rows < 1 || rows > 0x7fffffff) return "rows must be between 1 and 2^31 - 1";
    if (cols < (bin ? 0 : 1) || cols > (1 << 30)) return "cols must be between 1 (0 with a dustbin) and 2^30";
    if (ld < cols) return "the row stride is smaller than a row";
    if (!x) return "null argument";
    if ((uintptr_t)x & (dtype == IMP_DTYPE_F32 ? 3 : 1)) return "logits are not aligned to their type";
    return nullptr;
}
int ready(int device) {
    hipError_t e = hipSetDevice(device);
    return e == hipSuccess ? 0 : imp_fail(IMP_E_HIP, hipGetErrorString(e));
}

template <typename T, int K> void forward(const LogpOp& p, hipStream_t st) {
    if (p.shares == 1 && wave_rows(p.rows, p.cols)) logp_forward_kernel<T, K, 1><<<dim3((unsigned)((p.rows + 3) / 4), 1), 256, 0, st>>>(p);
    else logp_forward_kernel<T, K, 4><<<dim3((unsigned)p.rows, (unsigned)p.shares), 256, 0, st>>>(p);
    if (p.shares > 1) logp_join_kernel<T, K><<<(unsigned)((p.rows + 3) / 4), 256, 0, st>>>(p);
}
template <typename T> void forward_top(const LogpOp& p, hipStream_t st) {
    switch (padded_top(p.top)) {
        case 0: forward<T, 0>(p, st); break;
        case 1: forward<T, 1>(p, st); break;
        case 4: forward<T, 4>(p, st); break;
        case 8: forward<T, 8>(p, st); break;
        default: forward<T, TOP_MAX>(p, st);
    }
}
template <typename T> void backward(const LogpOp& p, hipStream_t st) {
    if (p.shares == 1 && wave_rows(p.rows, p.cols)) logp_backward_kernel<T, 1><<<dim3((unsigned)((p.rows + 3) / 4), 1), 256, 0, st>>>(p);
    else logp_backward_kernel<T, 4><<<dim3((unsigned)p.rows, (unsigned)p.shares), 256, 0, st>>>(p);
}

}  // namespace

extern "C" {

int imp_log_probs_workspace(int64_t rows, int cols, int top, int backward, uint64_t* bytes) {
    if (!bytes || rows < 1 || cols < 0 || top < 0 || top > TOP_MAX) return imp_fail(IMP_E_ARG, "imp_log_probs_workspace: bad argument");
    const int s = shares_of(rows, cols);
    if (backward) *bytes = (uint64_t)rows * 8;
    else *bytes = s > 1 ? (uint64_t)rows * s * (12 + 8 * padded_top(top)) : 0;
    return IMP_OK;
}

int imp_log_probs_forward(int dtype, int64_t rows, int cols, int64_t ld, const void* logits, const float* bin_score, const int64_t* targets, int top, float* logp,
                          float* entropy, float* stats, float* top_logp, int64_t* top_ids, void* workspace, uint64_t workspace_bytes, int device, void* stream) {
    if (const char* why = bad(dtype, rows, cols, ld, logits, bin_score != nullptr)) return imp_fail(IMP_E_ARG, why);
    if (top < 0 || top > TOP_MAX) return imp_fail(IMP_E_ARG, "top must be between 0 and 16");
    if (!targets || !logp || !entropy || !stats || (top && (!top_logp || !top_ids))) return imp_fail(IMP_E_ARG, "imp_log_probs_forward: null argument");
    uint64_t need = 0;
    imp_log_probs_workspace(rows, cols, top, 0, &need);
    if (workspace_bytes < need || (need && (!workspace || ((uintptr_t)workspace & 3)))) return imp_fail(IMP_E_NOMEM, "imp_log_probs_forward: workspace too small");
    if (int rc = ready(device)) return rc;
    LogpOp p = {};
    p.x = logits; p.target = targets; p.bin = bin_score; p.logp = logp; p.entropy = entropy; p.stats = stats; p.top_logp = top_logp; p.top_id = top_ids;
    p.rows = rows; p.ld = ld; p.cols = cols; p.top = top; p.shares = shares_of(rows, cols);
    p.part = (float*)workspace;
    p.part_v = p.part + 3 * rows * p.shares;
    p.part_i = (int*)(p.part_v + rows * p.shares * padded_top(top));
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == IMP_DTYPE_F32) forward_top<float>(p, st);
    else if (dtype == IMP_DTYPE_F16) forward_top<_Float16>(p, st);
    else forward_top<__bf16>(p, st);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? IMP_OK : imp_fail(IMP_E_HIP, hipGetErrorString(e));
}

int imp_log_probs_backward(int dtype, int64_t rows, int cols, int64_t ld, const void* logits, const float* bin_score, const int64_t* targets, const float* entropy,
                           const float* stats, const float* dlogp, const float* dentropy, void* dlogits, float* dbin, void* workspace,
                           uint64_t workspace_bytes, int device, void* stream) {
    if (const char* why = bad(dtype, rows, cols, ld, logits, bin_score != nullptr)) return imp_fail(IMP_E_ARG, why);
    if (!targets || !entropy || !stats || (!dlogits && !dbin) || (dbin && !bin_score)) return imp_fail(IMP_E_ARG, "imp_log_probs_backward: null argument");
    if ((uintptr_t)dlogits & (dtype == IMP_DTYPE_F32 ? 3 : 1)) return imp_fail(IMP_E_ARG, "dlogits are not aligned to their type");
    if (dbin && (workspace_bytes < (uint64_t)rows * 8 || !workspace || ((uintptr_t)workspace & 7)))
        return imp_fail(IMP_E_NOMEM, "imp_log_probs_backward: workspace too small");
    if (int rc = ready(device)) return rc;
    LogpOp p = {};
    p.x = logits; p.target = targets; p.bin = bin_score; p.entropy = const_cast<float*>(entropy); p.stats = const_cast<float*>(stats);
    p.dlogp = dlogp; p.dentropy = dentropy; p.dx = dlogits; p.rows = rows; p.ld = ld; p.cols = cols; p.shares = shares_of(rows, cols);
    p.part_bin = dbin ? (double*)workspace : nullptr;
    const hipStream_t st = (hipStream_t)stream;
    if (dtype == IMP_DTYPE_F32) backward<float>(p, st);
    else if (dtype == IMP_DTYPE_F16) backward<_Float16>(p, st);
    else backward<__bf16>(p, st);
    if (dbin) logp_bin_kernel<<<1, 1024, 0, st>>>(p.part_bin, rows, dbin);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? IMP_OK : imp_fail(IMP_E_HIP, hipGetErrorString(e));
}

}  // extern "C"
