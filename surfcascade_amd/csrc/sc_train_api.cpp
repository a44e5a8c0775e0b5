// sc_train_api.cpp -- the C ABI of the training side over a mined sample
// matrix (include/surfcascade.h sc_trainer_*, sc_lr_*, sc_sample): argument
// checks, stream order, workspaces, launches.
#include <hip/hip_runtime.h>

#include <climits>
#include <cmath>
#include <cstdlib>
#include <cstring>

#include "sc_host.hpp"
#include "sc_train.hpp"

using sc::check_device_ptr;
using sc::Error;
using sc::guarded;

struct sc_trainer {
    int device = 0;
    hipStream_t stream = nullptr;      // where launches go: own_stream, or the caller's
    hipStream_t own_stream = nullptr;  // created with the trainer, destroyed with it
    hipEvent_t event = nullptr;        // recorded and waited on at once (stream order)
    hipEvent_t left = nullptr;         // end of the stream last left for one under capture ...
    bool pending = false;              // ... whose work no later stream waits for yet
    sc::DevBuf<char> ws;               // workspace of calls that bring none

    ~sc_trainer() {
        int before = 0;
        (void)hipGetDevice(&before);
        (void)hipSetDevice(device);
        // (a caller's stream is not touched: freeing waits for the device)
        if (own_stream) (void)hipStreamSynchronize(own_stream);
        ws.release();
        if (left) (void)hipEventDestroy(left);
        if (event) (void)hipEventDestroy(event);
        if (own_stream) (void)hipStreamDestroy(own_stream);
        (void)hipSetDevice(before);
    }
};

namespace {

// the trainer's GPU for the length of a call; the caller's current device after
struct OnDevice {
    int before = 0;
    explicit OnDevice(int device) {
        HIPCHK(hipGetDevice(&before));
        if (before != device) HIPCHK(hipSetDevice(device));
        now = device;
    }
    ~OnDevice() {
        if (before != now) (void)hipSetDevice(before);
    }
    OnDevice(const OnDevice &) = delete;
    OnDevice &operator=(const OnDevice &) = delete;

   private:
    int now = 0;
};

void need(bool ok, const char *msg) {
    if (!ok) throw Error{SC_ERR_INVALID, msg};
}

void need_ptr(const sc_trainer *t, const void *p, const char *what, bool optional = false) {
    if (!p && !optional) throw Error{SC_ERR_INVALID, std::string(what) + " is NULL"};
    check_device_ptr(t->device, "trainer", p, what);
}

bool capturing(hipStream_t s) {
    if (!s) return false;  // the null stream cannot be captured
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    HIPCHK(hipStreamIsCapturing(s, &st));
    return st != hipStreamCaptureStatusNone;
}

// The trainer's stream waits for the one left before a capture, whose calls may
// still use the trainer's workspace.
void catch_up(sc_trainer *t) {
    if (!t->pending) return;
    HIPCHK(hipStreamWaitEvent(t->stream, t->left, 0));
    t->pending = false;
}

// `bytes` of workspace: the caller's, or the trainer's own.  Growing the own
// one frees what an earlier call may still use only after the device is idle
// (hipFree); inside a capture there is no growing, and two graphs must not
// share one, so a captured call brings its own.
void *workspace(sc_trainer *t, size_t bytes, void *ws, size_t ws_bytes) {
    if (bytes == 0) return nullptr;
    if (ws) {
        if (ws_bytes < bytes)
            throw Error{SC_ERR_CAPACITY, "workspace of " + std::to_string(ws_bytes) + " bytes, " +
                                             std::to_string(bytes) + " needed"};
        need((reinterpret_cast<uintptr_t>(ws) & 15) == 0, "workspace is not aligned to 16 bytes");
        need_ptr(t, ws, "workspace");
        return ws;
    }
    if (capturing(t->stream))
        throw Error{SC_ERR_INVALID, "a call under stream capture needs a workspace of its own"};
    catch_up(t);
    if (bytes > t->ws.n) HIPCHK(hipStreamSynchronize(t->stream));
    t->ws.ensure(bytes);
    return t->ws.p;
}

int elem_size(int dtype) { return dtype == SC_F32 ? 4 : 2; }

void need_aligned(const void *p, size_t size, const char *what) {
    if (reinterpret_cast<uintptr_t>(p) % size)
        throw Error{SC_ERR_INVALID, std::string(what) + " is not aligned to its elements"};
}

constexpr int64_t kMostRows = 1 << 30;  // row numbers and their steps stay in 32 bits

// every host-side check of the operands all sc_lr_* share
sc::LrArgs lr_args(const sc_samples *x, const sc_weak_bank *k) {
    need(x && k, "null argument");
    need(x->dtype == SC_F32 || x->dtype == SC_F16 || x->dtype == SC_BF16, "unknown sample type");
    need(x->n >= 0 && x->n <= kMostRows, "bad number of samples");
    need(x->n_patches >= 1 && x->n_patches <= (1 << 24), "bad number of patches");
    need(x->ld >= (int64_t)sc::kDesc * x->n_patches, "samples overlap (ld < 32 * n_patches)");
    need(x->ld <= ((int64_t)1 << 40), "bad sample stride");
    need(!x->rows || (x->n_rows >= 0 && x->n_rows <= kMostRows), "bad number of rows");
    need(k->m >= 0 && k->h >= 0 && k->h <= 1024, "bad number of weak learners");
    need((int64_t)k->m * k->h <= (1 << 25), "too many weak learners");
    need(k->patch || k->m <= x->n_patches, "more weak learners than patches and no patch numbers");
    sc::LrArgs a{};
    a.x = x->data;
    a.ld = x->ld;
    a.n = (int)x->n;
    a.n_patches = x->n_patches;
    a.dtype = x->dtype;
    a.rows = x->rows;
    a.R = (int)(x->rows ? x->n_rows : x->n);
    a.M = k->m;
    a.H = k->h;
    a.patch = k->patch;
    a.w = k->w;
    a.b = k->b;
    a.alpha = 1.0f;
    a.beta = 1.0f;
    if (a.n == 0) {  // every row is absent: what is read in their place lies in the weights
        a.x = a.w;
        a.ld = 0;
        a.n_patches = 0;
    }
    return a;
}

void lr_pointers(const sc_trainer *t, const sc::LrArgs &a) {
    if (a.M == 0 || a.H == 0) return;
    if (a.R > 0) {
        need_ptr(t, a.x, "samples");
        need_aligned(a.x, elem_size(a.dtype), "samples");
    }
    if (a.R > 0) need_ptr(t, a.rows, "rows", true);
    need_ptr(t, a.patch, "patch", true);
    need_ptr(t, a.w, "w");
    need_ptr(t, a.b, "b", true);
}

int lr_grad(sc_trainer *t, const sc::LrArgs &a, bool loss, void *ws, size_t ws_bytes) {
    const sc::LrPlan p = sc::lr_plan(a);
    sc::launch_lr_grad(a, p, workspace(t, p.acc_bytes + p.part_bytes, ws, ws_bytes), loss, t->stream);
    HIPCHK(hipGetLastError());
    return SC_OK;
}

}  // namespace

extern "C" {

int sc_trainer_create(int device, sc_trainer **out) {
    return guarded([&] {
        need(out, "null argument");
        int ndev = 0;
        HIPCHK(hipGetDeviceCount(&ndev));
        if (device < 0 || device >= ndev)
            throw Error{SC_ERR_DEVICE, "device " + std::to_string(device) + " not present (" +
                                           std::to_string(ndev) + " visible)"};
        hipDeviceProp_t prop;
        HIPCHK(hipGetDeviceProperties(&prop, device));
        if (std::strncmp(prop.gcnArchName, "gfx950", 6) != 0)
            throw Error{SC_ERR_DEVICE, std::string("kernels are built for gfx950, device is ") + prop.gcnArchName};
        OnDevice on(device);
        auto *t = new sc_trainer();
        try {
            t->device = device;
            HIPCHK(hipStreamCreateWithFlags(&t->own_stream, hipStreamNonBlocking));
            t->stream = t->own_stream;
            HIPCHK(hipEventCreateWithFlags(&t->event, hipEventDisableTiming));
            HIPCHK(hipEventCreateWithFlags(&t->left, hipEventDisableTiming));
        } catch (...) {
            delete t;
            throw;
        }
        *out = t;
        return SC_OK;
    });
}

void sc_trainer_destroy(sc_trainer *t) { delete t; }

void *sc_trainer_stream(sc_trainer *t) { return t ? (void *)t->stream : nullptr; }

int sc_trainer_wait_stream(sc_trainer *t, void *stream) {
    return guarded([&] {
        need(t, "null trainer");
        OnDevice on(t->device);
        HIPCHK(hipEventRecord(t->event, static_cast<hipStream_t>(stream)));
        HIPCHK(hipStreamWaitEvent(t->stream, t->event, 0));
        return SC_OK;
    });
}

int sc_stream_wait_trainer(sc_trainer *t, void *stream) {
    return guarded([&] {
        need(t, "null trainer");
        OnDevice on(t->device);
        HIPCHK(hipEventRecord(t->event, t->stream));
        HIPCHK(hipStreamWaitEvent(static_cast<hipStream_t>(stream), t->event, 0));
        return SC_OK;
    });
}

int sc_trainer_set_stream(sc_trainer *t, void *stream, int use_own) {
    return guarded([&] {
        need(t, "null trainer");
        OnDevice on(t->device);
        hipStream_t s = use_own ? t->own_stream : static_cast<hipStream_t>(stream);
        if (s == t->stream) return SC_OK;
        if (s && !use_own) {
            int dev = -1;
            HIPCHK(hipStreamGetDevice(s, &dev));
            if (dev != t->device)
                throw Error{SC_ERR_INVALID, "stream of device " + std::to_string(dev) + ", trainer on " +
                                                std::to_string(t->device)};
        }
        // an event may not tie a capturing stream to one outside the capture:
        // eager work then waits for eager work (a captured call has no part in
        // the trainer's workspace)
        if (!capturing(t->stream)) {
            catch_up(t);
            const bool to = capturing(s);
            HIPCHK(hipEventRecord(to ? t->left : t->event, t->stream));
            if (to) t->pending = true;
            else HIPCHK(hipStreamWaitEvent(s, t->event, 0));
        }
        t->stream = s;
        return SC_OK;
    });
}

int sc_trainer_synchronize(sc_trainer *t) {
    return guarded([&] {
        need(t, "null trainer");
        OnDevice on(t->device);
        HIPCHK(hipStreamSynchronize(t->stream));
        return SC_OK;
    });
}

int sc_lr_response(sc_trainer *t, const sc_samples *x, const sc_weak_bank *k, int act, float alpha,
                   const float *res, int res_kind, int64_t res_ld, float beta, float *y, int64_t y_ld) {
    return guarded([&] {
        sc::LrArgs a = lr_args(x, k);
        const int64_t cols = (int64_t)a.M * a.H;
        need(act == SC_ACT_NONE || act == SC_ACT_SIGMOID, "unknown activation");
        need(res_kind >= SC_RES_NONE && res_kind <= SC_RES_FULL, "unknown residual kind");
        need((res_kind != SC_RES_NONE) == (res != nullptr) || a.R == 0 || cols == 0, "residual and its kind disagree");
        need(y_ld >= cols, "y_ld smaller than a row of results");
        need(res_kind != SC_RES_FULL || res_ld >= cols, "res_ld smaller than a row of results");
        need(res_kind != SC_RES_ROW || res_ld >= 1, "bad res_ld");
        need(t, "null trainer");
        if (a.R == 0 || cols == 0) return SC_OK;
        OnDevice on(t->device);
        lr_pointers(t, a);
        need_ptr(t, y, "y");
        need_ptr(t, res, "residual", true);
        a.act = act;
        a.alpha = alpha;
        a.beta = beta;
        a.res = res;
        a.res_kind = res_kind;
        a.res_ld = res_ld;
        a.y = y;
        a.y_ld = y_ld;
        sc::launch_lr_response(a, t->stream);
        HIPCHK(hipGetLastError());
        return SC_OK;
    });
}

int sc_lr_workspace(const sc_samples *x, const sc_weak_bank *k, size_t *bytes) {
    return guarded([&] {
        need(bytes, "null argument");
        const sc::LrArgs a = lr_args(x, k);
        const sc::LrPlan p = sc::lr_plan(a);
        *bytes = p.acc_bytes + p.part_bytes;
        return SC_OK;
    });
}

int sc_lr_response_grad(sc_trainer *t, const sc_samples *x, const sc_weak_bank *k, int act, float alpha,
                        const float *dy, int64_t dy_ld, float *dw, float *db, int res_kind, float beta,
                        float *dres, int64_t dres_ld, void *ws, size_t ws_bytes) {
    return guarded([&] {
        sc::LrArgs a = lr_args(x, k);
        const int64_t cols = (int64_t)a.M * a.H;
        need(act == SC_ACT_NONE || act == SC_ACT_SIGMOID, "unknown activation");
        need(res_kind >= SC_RES_NONE && res_kind <= SC_RES_FULL, "unknown residual kind");
        need((res_kind != SC_RES_NONE) == (dres != nullptr) || a.R == 0 || (cols == 0 && res_kind != SC_RES_ROW),
             "dres and its kind disagree");
        need(dy_ld >= cols, "dy_ld smaller than a row of results");
        need(res_kind != SC_RES_FULL || dres_ld >= cols, "dres_ld smaller than a row of results");
        need(res_kind != SC_RES_ROW || dres_ld >= 1, "bad dres_ld");
        need(t, "null trainer");
        OnDevice on(t->device);
        lr_pointers(t, a);
        if (a.R > 0 && cols > 0) need_ptr(t, dy, "dy");
        if (cols > 0) {
            need_ptr(t, dw, "dw");
            need_ptr(t, db, "db");
        }
        need_ptr(t, dres, "dres", true);
        a.act = act;
        a.alpha = alpha;
        a.beta = beta;
        a.dy = dy;
        a.dy_ld = dy_ld;
        a.dw = dw;
        a.db = db;
        a.res_kind = res_kind;
        a.dres = dres;
        a.dres_ld = dres_ld;
        if (cols == 0 && res_kind != SC_RES_ROW) return SC_OK;
        lr_grad(t, a, false, ws, ws_bytes);
        return SC_OK;
    });
}

int sc_lr_loss(sc_trainer *t, const sc_samples *x, const sc_weak_bank *k, const float *target,
               const float *weight, float *loss, float *dw, float *db, void *ws, size_t ws_bytes) {
    return guarded([&] {
        sc::LrArgs a = lr_args(x, k);
        need(t, "null trainer");
        if (a.M == 0 || a.H == 0) return SC_OK;
        OnDevice on(t->device);
        lr_pointers(t, a);
        if (a.R > 0 && a.n > 0) need_ptr(t, target, "target");
        need_ptr(t, weight, "weight", true);
        need_ptr(t, loss, "loss");
        need_ptr(t, dw, "dw");
        need_ptr(t, db, "db");
        a.target = target;
        a.weight = weight;
        a.loss = loss;
        a.dw = dw;
        a.db = db;
        return lr_grad(t, a, true, ws, ws_bytes);
    });
}

void sc_sample_params_default(sc_sample_params *p) {
    if (!p) return;
    p->temperature = 1.0;
    p->top_k = 0;
    p->top_p = 1.0;
    p->min_p = 0.0;
}

int sc_sample_workspace(int b, int v, int s, size_t *bytes) {
    return guarded([&] {
        need(bytes, "null argument");
        need(b >= 0 && v >= 0 && s >= 0, "negative size");
        need(v <= sc::kMaxPool, "more than 2^26 scores in a row");
        need(b <= kMostRows && s <= kMostRows, "more than 2^30 rows or draws");
        sc::SampleArgs a{};
        a.B = b;
        a.V = v;
        a.S = s;
        a.temperature = 1.0;  // (no trim: the most any parameters need)
        a.top_p = 1.0;
        *bytes = sc::sample_plan(a).ws_bytes;
        return SC_OK;
    });
}

int sc_sample(sc_trainer *t, const void *scores, int dtype, int b, int v, int64_t ld, const int32_t *lens,
              const sc_sample_params *prm, const double *u, int s, int64_t u_ld, int32_t *index,
              int64_t index_ld, int32_t *kept, void *ws, size_t ws_bytes) {
    return guarded([&] {
        sc_sample_params p;
        if (prm) p = *prm;
        else sc_sample_params_default(&p);
        need(dtype == SC_F32 || dtype == SC_F16 || dtype == SC_BF16, "unknown score type");
        need(b >= 0 && v >= 0 && s >= 0, "negative size");
        need(v <= sc::kMaxPool, "more than 2^26 scores in a row");
        need(b <= kMostRows && s <= kMostRows, "more than 2^30 rows or draws");
        need(ld >= v || b <= 1, "rows of scores overlap (ld < v)");
        need(u_ld >= s || b <= 1, "rows of u overlap");
        need(index_ld >= s || b <= 1, "rows of index overlap");
        need(p.temperature >= 0.0 && std::isfinite(p.temperature), "temperature must be finite and >= 0");
        need(p.top_k >= 0, "top_k must be >= 0 (0: off)");
        need(p.top_p >= 0.0, "top_p must be >= 0 (1: off)");
        need(p.min_p >= 0.0 && p.min_p <= 1.0, "min_p must be in [0, 1]");
        need(t, "null trainer");
        if (b == 0) return SC_OK;
        OnDevice on(t->device);
        if (v > 0) {
            need_ptr(t, scores, "scores");
            need_aligned(scores, elem_size(dtype), "scores");
        }
        need_ptr(t, lens, "lens", true);
        if (s > 0) {
            need_ptr(t, u, "u");
            need_ptr(t, index, "index");
        }
        need_ptr(t, kept, "kept", true);
        sc::SampleArgs a{};
        a.scores = scores;
        a.dtype = dtype;
        a.B = b;
        a.V = v;
        a.ld = ld;
        a.lens = lens;
        a.temperature = p.temperature;
        a.top_k = p.top_k;
        a.top_p = p.top_p;
        a.min_p = p.min_p;
        a.shift = sc::sample_shift(v);
        a.u = u;
        a.S = s;
        a.u_ld = u_ld;
        a.index = index;
        a.index_ld = index_ld;
        a.kept = kept;
        a.ws = workspace(t, sc::sample_plan(a).ws_bytes, ws, ws_bytes);
        sc::launch_sample(a, t->stream);
        HIPCHK(hipGetLastError());
        return SC_OK;
    });
}

}  // extern "C"
