// gated_scan.cu -- the gated linear recurrence h_t = c_t h_{t-1} + (1 - a_t) x_t with
// a = sigmoid(gate), forward, backward and single step.  One thread per (batch row,
// channel) walks the sequence; the backward pass forms the states of one block of
// DG_SCAN_MARK_STEPS steps again from its mark before walking the block in reverse.
#include "lm_common.cuh"

namespace {

struct ScanIn {
    const void *x, *g, *o;
    int64_t x_sb, x_st, g_sb, g_st, o_sb, o_st;
    const int32_t* lengths;
    const uint8_t* resets;
    int B, T, D;
};

template <typename T>
__global__ void scan_forward_kernel(ScanIn in, const float* h0, T* y, float* h_last, float* marks) {
    const int d = blockIdx.x * blockDim.x + threadIdx.x, b = blockIdx.y;
    if (d >= in.D) return;
    const T* x = (const T*)in.x + b * in.x_sb + d;
    const T* g = (const T*)in.g + b * in.g_sb + d;
    const T* o = in.o ? (const T*)in.o + b * in.o_sb + d : nullptr;
    const int nblk = (in.T + DG_SCAN_MARK_STEPS - 1) / DG_SCAN_MARK_STEPS;
    const int len = in.lengths ? min(max(in.lengths[b], 0), in.T) : in.T;
    float h = h0 ? h0[(int64_t)b * in.D + d] : 0.f;
    for (int t = 0; t < in.T; ++t) {
        if (marks && t % DG_SCAN_MARK_STEPS == 0)
            marks[((int64_t)b * nblk + t / DG_SCAN_MARK_STEPS) * in.D + d] = h;
        float out = 0.f;
        if (t < len) {
            float a, na;
            dg::sigmoid_pair(dg::to_f(g[t * in.g_st]), a, na);
            const float c = (in.resets && in.resets[(int64_t)b * in.T + t]) ? 0.f : a;
            h = fmaf(c, h, na * dg::to_f(x[t * in.x_st]));
            out = h;
            if (o) {
                const float z = dg::to_f(o[t * in.o_st]);
                out = h * (z * dg::sigmoid(z));
            }
        }
        y[((int64_t)b * in.T + t) * in.D + d] = dg::from_f<T>(out);
    }
    if (h_last) h_last[(int64_t)b * in.D + d] = h;
}

struct ScanGrad {
    const float* marks;
    const void* dy;
    int64_t dy_sb, dy_st;
    const float* dh_last;
    void *dx, *dg_, *do_;
    int64_t dx_sb, dx_st, dg_sb, dg_st, do_sb, do_st;
    float* dh0;
};

constexpr int BW_THREADS = 64;

template <typename T>
__global__ void scan_backward_kernel(ScanIn in, ScanGrad q) {
    __shared__ float hs[DG_SCAN_MARK_STEPS][BW_THREADS];       // the state before each step of the block
    const int d = blockIdx.x * blockDim.x + threadIdx.x, b = blockIdx.y, me = threadIdx.x;
    if (d >= in.D) return;
    const T* x = (const T*)in.x + b * in.x_sb + d;
    const T* g = (const T*)in.g + b * in.g_sb + d;
    const T* o = in.o ? (const T*)in.o + b * in.o_sb + d : nullptr;
    const T* dy = (const T*)q.dy + b * q.dy_sb + d;
    T* dx = (T*)q.dx + b * q.dx_sb + d;
    T* dgt = (T*)q.dg_ + b * q.dg_sb + d;
    T* dot = in.o ? (T*)q.do_ + b * q.do_sb + d : nullptr;
    const int nblk = (in.T + DG_SCAN_MARK_STEPS - 1) / DG_SCAN_MARK_STEPS;
    const int len = in.lengths ? min(max(in.lengths[b], 0), in.T) : in.T;
    const uint8_t* rs = in.resets ? in.resets + (int64_t)b * in.T : nullptr;
    float e = q.dh_last ? q.dh_last[(int64_t)b * in.D + d] : 0.f;    // c_{t+1} e_{t+1}
    for (int blk = nblk - 1; blk >= 0; --blk) {
        const int t0 = blk * DG_SCAN_MARK_STEPS, t1 = min(t0 + DG_SCAN_MARK_STEPS, in.T);
        float h = q.marks[((int64_t)b * nblk + blk) * in.D + d];
        for (int t = t0; t < min(t1, len); ++t) {
            hs[t - t0][me] = h;
            float a, na;
            dg::sigmoid_pair(dg::to_f(g[t * in.g_st]), a, na);
            h = fmaf((rs && rs[t]) ? 0.f : a, h, na * dg::to_f(x[t * in.x_st]));
        }
        for (int t = t1 - 1; t >= t0; --t) {
            float rx = 0.f, rg = 0.f, ro = 0.f;
            if (t < len) {
                float a, na;
                dg::sigmoid_pair(dg::to_f(g[t * in.g_st]), a, na);
                const float keep = (rs && rs[t]) ? 0.f : 1.f;
                const float xt = dg::to_f(x[t * in.x_st]), hp = keep * hs[t - t0][me];
                const float dyt = dg::to_f(dy[t * q.dy_st]);
                float gate = 1.f;
                if (o) {
                    const float z = dg::to_f(o[t * in.o_st]);
                    float s, n;
                    dg::sigmoid_pair(z, s, n);
                    gate = z * s;
                    ro = dyt * fmaf(a, hp, na * xt) * (s * fmaf(z, n, 1.f));
                }
                e = fmaf(dyt, gate, e);
                rx = e * na;
                rg = e * (hp - xt) * (a * na);
                e *= keep * a;
            }
            dx[t * q.dx_st] = dg::from_f<T>(rx);
            dgt[t * q.dg_st] = dg::from_f<T>(rg);
            if (o) dot[t * q.do_st] = dg::from_f<T>(ro);
        }
    }
    if (q.dh0) q.dh0[(int64_t)b * in.D + d] = e;
}

template <typename T>
__global__ void scan_step_kernel(int D, const T* x, int64_t x_sb, const T* g, int64_t g_sb, const T* o, int64_t o_sb,
                                 float* h, T* y) {
    const int d = blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t b = blockIdx.y;
    if (d >= D) return;
    float a, na;
    dg::sigmoid_pair(dg::to_f(g[b * g_sb + d]), a, na);
    const float hn = fmaf(a, h[b * D + d], na * dg::to_f(x[b * x_sb + d]));
    h[b * D + d] = hn;
    float out = hn;
    if (o) {
        const float z = dg::to_f(o[b * o_sb + d]);
        out = hn * (z * dg::sigmoid(z));
    }
    y[b * D + d] = dg::from_f<T>(out);
}

}  // namespace

extern "C" {

int dg_gated_scan_forward(int dtype, int B, int T, int D, const void* x, int64_t x_sb, int64_t x_st,
                          const void* gate, int64_t gate_sb, int64_t gate_st, const void* out_gate,
                          int64_t out_gate_sb, int64_t out_gate_st, const float* h0, const int32_t* lengths,
                          const uint8_t* resets, void* y, float* h_last, float* marks, void* stream) {
    if (dtype == DG_DTYPE_F64) return DG_ERR_UNSUPPORTED;
    if (dtype < DG_DTYPE_F32 || dtype > DG_DTYPE_BF16 || B < 0 || T < 0 || D < 0) return DG_ERR_INVALID_ARGUMENT;
    if (B == 0 || D == 0) return DG_OK;
    if (T > 0 && (!x || !gate || !y)) return DG_ERR_INVALID_ARGUMENT;
    if (T == 0 && !h_last) return DG_OK;
    if (B > 65535) return DG_ERR_UNSUPPORTED;                  // grid.y limit
    const ScanIn in{x, gate, out_gate, x_sb, x_st, gate_sb, gate_st, out_gate_sb, out_gate_st, lengths, resets, B, T, D};
    DG_DISPATCH_LM(dtype, S, {
        scan_forward_kernel<S><<<dim3((D + 63) / 64, B), 64, 0, static_cast<cudaStream_t>(stream)>>>(
            in, h0, static_cast<S*>(y), h_last, marks);
    });
    return dg_host::check_launch();
}

int dg_gated_scan_backward(int dtype, int B, int T, int D, const void* x, int64_t x_sb, int64_t x_st,
                           const void* gate, int64_t gate_sb, int64_t gate_st, const void* out_gate,
                           int64_t out_gate_sb, int64_t out_gate_st, const int32_t* lengths, const uint8_t* resets,
                           const float* marks, const void* dy, int64_t dy_sb, int64_t dy_st, const float* dh_last,
                           void* dx, int64_t dx_sb, int64_t dx_st, void* dgate, int64_t dgate_sb, int64_t dgate_st,
                           void* dout_gate, int64_t dout_gate_sb, int64_t dout_gate_st, float* dh0, void* stream) {
    if (dtype == DG_DTYPE_F64) return DG_ERR_UNSUPPORTED;
    if (dtype < DG_DTYPE_F32 || dtype > DG_DTYPE_BF16 || B < 0 || T < 0 || D < 0) return DG_ERR_INVALID_ARGUMENT;
    if ((out_gate == nullptr) != (dout_gate == nullptr)) return DG_ERR_INVALID_ARGUMENT;
    if (B == 0 || D == 0) return DG_OK;
    if (T > 0 && (!x || !gate || !marks || !dy || !dx || !dgate)) return DG_ERR_INVALID_ARGUMENT;
    if (T == 0 && !dh0) return DG_OK;
    if (B > 65535) return DG_ERR_UNSUPPORTED;
    const ScanIn in{x, gate, out_gate, x_sb, x_st, gate_sb, gate_st, out_gate_sb, out_gate_st, lengths, resets, B, T, D};
    const ScanGrad q{marks, dy, dy_sb, dy_st, dh_last, dx, dgate, dout_gate, dx_sb, dx_st, dgate_sb, dgate_st,
                     dout_gate_sb, dout_gate_st, dh0};
    DG_DISPATCH_LM(dtype, S, {
        scan_backward_kernel<S><<<dim3((D + BW_THREADS - 1) / BW_THREADS, B), BW_THREADS, 0,
                                  static_cast<cudaStream_t>(stream)>>>(in, q);
    });
    return dg_host::check_launch();
}

int dg_gated_scan_step(int dtype, int B, int D, const void* x, int64_t x_sb, const void* gate, int64_t gate_sb,
                       const void* out_gate, int64_t out_gate_sb, float* h, void* y, void* stream) {
    if (dtype == DG_DTYPE_F64) return DG_ERR_UNSUPPORTED;
    if (dtype < DG_DTYPE_F32 || dtype > DG_DTYPE_BF16 || B < 0 || D < 0) return DG_ERR_INVALID_ARGUMENT;
    if (B == 0 || D == 0) return DG_OK;
    if (!x || !gate || !h || !y) return DG_ERR_INVALID_ARGUMENT;
    if (B > 65535) return DG_ERR_UNSUPPORTED;
    DG_DISPATCH_LM(dtype, S, {
        scan_step_kernel<S><<<dim3((D + 127) / 128, B), 128, 0, static_cast<cudaStream_t>(stream)>>>(
            D, static_cast<const S*>(x), x_sb, static_cast<const S*>(gate), gate_sb, static_cast<const S*>(out_gate),
            out_gate_sb, h, static_cast<S*>(y));
    });
    return dg_host::check_launch();
}

}  // extern "C"
