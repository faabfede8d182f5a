// cache_test.cpp - the paged cache and its attention through the C++ host layer (include/cybq.hpp).
//
//   cache_test --refusals   no GPU: what a backend without a device answers
//   cache_test --run        GPU: two sequences into an F16 cache in chunks, read back, attended to; compared with sums in double
//
// --run prints the largest error of y in units of its bound: y is off by its own rounding (2^-11 |y|) and by p, rounded to f16
// before the product with the values (2^-11 sum p |v|), and fp32 sums (taken as 2^-18 sum p |v|).
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdio>
#include <cstring>
#include <vector>

#include "cybq.hpp"

static void* to_device(const void* from, size_t bytes)
{
    void* p = nullptr;
    if (hipMalloc(&p, bytes) != hipSuccess || hipMemcpy(p, from, bytes, hipMemcpyHostToDevice) != hipSuccess) return nullptr;
    return p;
}

int main(int argc, char** argv)
{
    if (argc < 2) { std::fprintf(stderr, "usage: cache_test --refusals|--run\n"); return 2; }
    cybq::Backend be(0);
    if (!std::strcmp(argv[1], "--refusals")) {
        cybq::Cache none;
        cybq_batch batch{};
        const bool made = (bool)be.make_cache(CYBQ_CACHE_F16, 1, 1, 80, 32, 1, none);
        std::printf("made %d held %d read %d attention %d\n", made, (bool)none, be.cache_read(none, 0, batch, nullptr, nullptr, CYBQ_F16).code,
                    be.attention(none, 0, batch, nullptr, 0, CYBQ_F16, 1, 1.f, 0, nullptr).code);
        return 0;
    }
    if (!be.ok()) { std::printf("ERROR %d %s\n", be.status().code, be.status().text.c_str()); return 1; }
    const int H = 4, KV = 2, D = 64, P = 32, PAGES = 5, len[2] = {45, 70}, table[2][3] = {{4, 1, -1}, {0, 3, 2}};
    const int total = 115;
    std::vector<_Float16> q(total * H * D), k(total * KV * D), v(total * KV * D), k2(k.size()), v2(v.size()), y(q.size());
    uint32_t r = 12345;
    auto next = [&] { r = r * 1664525u + 1013904223u; return (_Float16)(((int)(r >> 16) - 32768) / 16384.0f); };
    for (auto& x : q) x = next();
    for (auto& x : k) x = next();
    for (auto& x : v) x = next();
    cybq::Cache cache;
    cybq::Status s = be.make_cache(CYBQ_CACHE_F16, 2, KV, D, P, PAGES, cache);
    if (!s) { std::printf("ERROR %d %s\n", s.code, s.text.c_str()); return 1; }
    cybq::Cache moved(std::move(cache));
    const int starts[3] = {0, len[0], total};
    void *dq = to_device(q.data(), q.size() * 2), *dk = to_device(k.data(), k.size() * 2), *dv = to_device(v.data(), v.size() * 2),
         *dqo = to_device(q.data(), q.size() * 2), *dk2 = to_device(k2.data(), k2.size() * 2), *dv2 = to_device(v2.data(), v2.size() * 2),
         *dy = to_device(y.data(), y.size() * 2);
    cybq_batch batch{2, total, 70, 3, (const int32_t*)to_device(starts, sizeof starts), (const int32_t*)to_device(len, sizeof len),
                     (const int32_t*)to_device(table, sizeof table)};
    if (!dq || !dk || !dv || !dqo || !dk2 || !dv2 || !dy || !batch.starts || !batch.lengths || !batch.tables) return 1;
    s = be.cache_append(moved, 1, batch, dq, H * D, H, dk, KV * D, dv, KV * D, CYBQ_F16, nullptr, 0, 0, CYBQ_ROPE_HALVES, dqo, CYBQ_F16);
    if (s) s = be.cache_read(moved, 1, batch, dk2, dv2, CYBQ_F16);
    if (s) s = be.attention(moved, 1, batch, dqo, H * D, CYBQ_F16, H, 0.125f, 0, dy);
    if (!s) { std::printf("ERROR %d %s\n", s.code, s.text.c_str()); return 1; }
    if (hipDeviceSynchronize() != hipSuccess || hipMemcpy(k2.data(), dk2, k2.size() * 2, hipMemcpyDeviceToHost) != hipSuccess ||
        hipMemcpy(v2.data(), dv2, v2.size() * 2, hipMemcpyDeviceToHost) != hipSuccess || hipMemcpy(y.data(), dy, y.size() * 2, hipMemcpyDeviceToHost) != hipSuccess)
        return 1;
    const bool same = !std::memcmp(k.data(), k2.data(), k.size() * 2) && !std::memcmp(v.data(), v2.data(), v.size() * 2);
    double worst = 0;
    for (int b = 0, t0 = 0; b < 2; t0 += len[b++])
        for (int i = 0; i < len[b]; i++)
            for (int h = 0; h < H; h++) {
                std::vector<double> p(i + 1);
                double top = -1e300, sum = 0;
                for (int j = 0; j <= i; j++) {
                    double dot = 0;
                    for (int d = 0; d < D; d++) dot += (double)q[((t0 + i) * H + h) * D + d] * (double)k[((t0 + j) * KV + h / 2) * D + d];
                    p[j] = dot * 0.125;
                    top = std::fmax(top, p[j]);
                }
                for (auto& e : p) sum += e = std::exp(e - top);
                for (int d = 0; d < D; d++) {
                    double want = 0, size = 0;
                    for (int j = 0; j <= i; j++) {
                        const double x = p[j] / sum * (double)v[((t0 + j) * KV + h / 2) * D + d];
                        want += x;
                        size += std::fabs(x);
                    }
                    const double bound = std::ldexp(std::fabs(want) + size, -11) + std::ldexp(size, -18) + std::ldexp(1.0, -24);
                    worst = std::fmax(worst, std::fabs((double)y[((t0 + i) * H + h) * D + d] - want) / bound);
                }
            }
    std::printf("stored %s worst %.3f\n", same ? "same" : "DIFFERENT", worst);
    for (void* p : {dq, dk, dv, dqo, dk2, dv2, dy, (void*)batch.starts, (void*)batch.lengths, (void*)batch.tables}) (void)hipFree(p);
    return same && worst <= 1.0 ? 0 : 1;
}
