// The training side through the C++ facade: two draws with replacement from a
// pool on the GPU, then the drawn rows' loss.  argv[1] "refuse": no GPU needed.
#include <hip/hip_runtime_api.h>

#include <cmath>
#include <cstdio>
#include <cstring>
#include <vector>

#include "surfcascade.hpp"

template <class T>
static T *to_gpu(const std::vector<T> &v) {
    void *p = nullptr;
    if (hipMalloc(&p, v.size() * sizeof(T)) != hipSuccess) return nullptr;
    if (hipMemcpy(p, v.data(), v.size() * sizeof(T), hipMemcpyHostToDevice) != hipSuccess) return nullptr;
    return static_cast<T *>(p);
}

int main(int argc, char **argv) {
    if (argc > 1 && !std::strcmp(argv[1], "refuse")) {
        size_t bytes = 1;
        sc_samples x{};
        sc_weak_bank k{};
        x.n_patches = 4;
        x.ld = 127;  // the samples would overlap
        std::printf("%d %s\n", sc_lr_workspace(&x, &k, &bytes), sc_last_error());
        return 0;
    }
    try {
        surfcascade::Trainer t(0);
        const int n = 3, p = 2;
        std::vector<float> x(n * p * 32, 0.0f), w(p * 32, 0.0f), out(p * 34);
        for (int i = 0; i < n; i++)
            for (int j = 0; j < p; j++) x[(i * p + j) * 32 + i] = 1.0f;
        std::vector<float> scores = {0.0f, -INFINITY, 0.0f}, target = {1.0f, 0.0f, 0.0f};
        std::vector<double> u = {0.25, 0.75};
        std::vector<int32_t> index(2, 7);
        int32_t *d_index = to_gpu(index);
        float *d_x = to_gpu(x), *d_w = to_gpu(w), *d_s = to_gpu(scores), *d_t = to_gpu(target), *d_o = to_gpu(out);
        double *d_u = to_gpu(u);
        t.Sample(d_s, SC_F32, 1, n, n, d_u, 2, d_index);
        sc_samples sx{d_x, SC_F32, p, n, p * 32, d_index, 2};
        sc_weak_bank k{p, 1, nullptr, d_w, nullptr};
        t.Loss(sx, k, d_t, nullptr, d_o, d_o + p, d_o + p * 33);
        t.Synchronize();
        if (hipMemcpy(index.data(), d_index, 8, hipMemcpyDeviceToHost) != hipSuccess) return 2;
        if (hipMemcpy(out.data(), d_o, out.size() * 4, hipMemcpyDeviceToHost) != hipSuccess) return 2;
        std::printf("drawn %d %d\nloss %.9g %.9g\ndw %g %g %g\ndb %g\n", index[0], index[1], out[0], out[1], out[p],
                    out[p + 1], out[p + 2], out[p * 33]);
    } catch (const surfcascade::Error &e) {
        std::printf("error %d\n", e.code);
        return 3;
    }
    return 0;
}
