// Layer norm's kernels with a row whose copies are never issued: what a wait that runs out leaves behind.  Compiled and run by
// test_gpu_norm_waits.py; prints a line per form and returns 0 where everything is as it has to be.
#include <cmath>
#include <cstdio>
#include <vector>

#include "../aristos_b200/csrc/layer_norm.cuh"

using namespace kleos;
using T = __half;

__device__ int g_lost;  // the row, -1 for none

namespace kleos {
namespace norm {
template <>
__device__ __forceinline__ void Ring<T, 1>::issue(long long r, int s) const {
    if (r >= total || r == g_lost) return;
    tc::mbar_expect_tx(&full[s], H * 2);
    tc::bulk_load(rows + s * H, from[0] + r * ld[0], H * 2, &full[s]);
}
template <>
__device__ __forceinline__ void Ring<T, 2>::issue(long long r, int s) const {
    if (r >= total || r == g_lost) return;
    tc::mbar_expect_tx(&full[s], 2 * H * 2);
    for (int m = 0; m < 2; ++m) tc::bulk_load(rows + (s * 2 + m) * H, from[m] + r * ld[m], H * 2, &full[s]);
}
}  // namespace norm
}  // namespace kleos

constexpr int kRows = 203, kBlocks = 3, kDepth = 2, kLost = 70;
constexpr long long kWait = 20000000;  // about ten milliseconds

template <typename E>
struct Buffer {
    E* p = nullptr;
    size_t n;
    explicit Buffer(size_t n_) : n(n_) { cudaMalloc(&p, n * sizeof(E)); }
    ~Buffer() { cudaFree(p); }
    void set(const std::vector<E>& v) { cudaMemcpy(p, v.data(), n * sizeof(E), cudaMemcpyHostToDevice); }
    std::vector<E> get() const {
        std::vector<E> v(n);
        cudaMemcpy(v.data(), p, n * sizeof(E), cudaMemcpyDeviceToHost);
        return v;
    }
};
void lose(int row) { cudaMemcpyToSymbol(g_lost, &row, sizeof row); }
bool same(float a, float b) { return a == b || (a != a && b != b); }

struct Result {
    std::vector<T> out;
    std::vector<float> a, b;  // mean and rstd; sums for dw and db
};
// Rows of group `group` of block `block` from the lost one on.
bool gone(int r, int groups) {
    const int step = kBlocks * groups;
    return r >= kLost && (r - kLost) % step == 0;
}

template <int G, int N>
Result forward(int H, int lost, const Buffer<T>& x) {
    constexpr int P = norm::kForwardGroups<G>;
    Buffer<T> y((size_t)kRows * H);
    Buffer<float> mean(kRows), rstd(kRows);
    norm::Args a{};
    a.x = x.p; a.y = y.p; a.mean = mean.p; a.rstd = rstd.p;
    a.ldx = a.ldy = a.H = H; a.rows = kRows; a.depth = kDepth; a.wait_cycles = kWait; a.eps = 1e-5f;
    lose(lost);
    const size_t smem = (size_t)P * kDepth * H * 2;
    cudaFuncSetAttribute(norm::forward_kernel<T, 8, G, N>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    norm::forward_kernel<T, 8, G, N><<<kBlocks, G * P, smem>>>(a);
    cudaDeviceSynchronize();
    return Result{y.get(), mean.get(), rstd.get()};
}
template <int G, int N>
Result backward(int H, int lost, const Buffer<T>& x, const Buffer<T>& dy, const Buffer<float>& mean, const Buffer<float>& rstd) {
    constexpr int P = norm::kGroups<G>;
    Buffer<T> dx((size_t)kRows * H);
    Buffer<float> partial((size_t)kBlocks * 2 * H);
    norm::Args a{};
    a.x = x.p; a.dy = dy.p; a.dx = dx.p; a.mean = mean.p; a.rstd = rstd.p; a.partial = partial.p;
    a.ldx = a.lddy = a.lddx = a.H = H; a.rows = kRows; a.depth = kDepth; a.wait_cycles = kWait;
    lose(lost);
    const size_t smem = (size_t)(H * 4 + 127) / 128 * 128 + std::max((size_t)P * kDepth * 2 * H * 2, (size_t)8 * H * P);
    cudaFuncSetAttribute(norm::backward_kernel<T, 8, G, N>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    norm::backward_kernel<T, 8, G, N><<<kBlocks, G * P, smem>>>(a);
    cudaDeviceSynchronize();
    return Result{dx.get(), partial.get(), {}};
}

bool finite(const Result& r) {
    bool ok = true;
    for (const T v : r.out) ok = ok && std::isfinite(__half2float(v));
    for (const float v : r.a) ok = ok && std::isfinite(v);
    for (const float v : r.b) ok = ok && std::isfinite(v);
    return ok;
}

template <int GF, int NF, int GB, int NB>
int form(int H_forward, int H_back) {
    int wrong = 0;
    auto fill = [](size_t n, unsigned seed) {
        std::vector<T> v(n);
        for (T& e : v) {
            seed = seed * 1664525u + 1013904223u;
            e = __float2half((float)(seed >> 8) / (1 << 23) - 1.f);
        }
        return v;
    };
    {
        Buffer<T> x((size_t)kRows * H_forward);
        x.set(fill(x.n, 1));
        const Result whole = forward<GF, NF>(H_forward, -1, x), cut = forward<GF, NF>(H_forward, kLost, x);
        if (!finite(whole)) ++wrong;
        for (int r = 0; r < kRows; ++r) {
            const bool lost = gone(r, norm::kForwardGroups<GF>);
            auto right = [&](float w, float c) { return lost ? c != c : same(w, c); };
            if (!right(whole.a[r], cut.a[r]) || !right(whole.b[r], cut.b[r])) ++wrong;
            for (int j = 0; j < H_forward; ++j)
                if (!right(__half2float(whole.out[(size_t)r * H_forward + j]), __half2float(cut.out[(size_t)r * H_forward + j]))) ++wrong;
        }
        std::printf("forward %d: %d wrong\n", H_forward, wrong);
    }
    const int before = wrong;
    {
        const int H = H_back;
        Buffer<T> x((size_t)kRows * H), dy((size_t)kRows * H);
        x.set(fill(x.n, 2));
        dy.set(fill(dy.n, 3));
        Buffer<float> mean(kRows), rstd(kRows);
        mean.set(std::vector<float>(kRows, 0.01f));
        rstd.set(std::vector<float>(kRows, 1.7f));
        const Result whole = backward<GB, NB>(H, -1, x, dy, mean, rstd), cut = backward<GB, NB>(H, kLost, x, dy, mean, rstd);
        if (!finite(whole)) ++wrong;
        for (int r = 0; r < kRows; ++r)
            for (int j = 0; j < H; ++j) {
                const float w = __half2float(whole.out[(size_t)r * H + j]), c = __half2float(cut.out[(size_t)r * H + j]);
                if (!(gone(r, norm::kGroups<GB>) ? c != c : same(w, c))) ++wrong;
            }
        for (int block = 0; block < kBlocks; ++block)  // both sums of every column of the block that lost a row
            for (int j = 0; j < 2 * H; ++j) {
                const float w = whole.a[(size_t)block * 2 * H + j], c = cut.a[(size_t)block * 2 * H + j];
                if (!(block == kLost % kBlocks ? c != c : same(w, c))) ++wrong;
            }
        std::printf("gradients %d: %d wrong\n", H, wrong - before);
    }
    return wrong;
}

int main() {
    const int wrong = form<32, 1, 32, 2>(256, 512) + form<128, 3, 128, 2>(2880, 2048) + form<256, 2, 256, 3>(4096, 5120);
    const cudaError_t e = cudaGetLastError();
    std::printf("%s\n", cudaGetErrorString(e));
    return wrong == 0 && e == cudaSuccess ? 0 : 1;
}
