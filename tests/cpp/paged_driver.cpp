// paged_driver.cpp -- PagedKVCache (libinferno.so) on given queries, keys and values, without a model.
//
//   paged_driver <dir> <f32|bf16> <groups> <beams> <layers> <H> <D> <prompt> <steps> <page> <capacity> <budget> <recent>
//       reads the prompt's q.bin k.bin v.bin ([layers, groups, H, prompt, D]), the steps' sq.bin sk.bin sv.bin
//       ([steps, layers, groups * beams, H, 1, D]), all fp32, and with beams > 1 parents.bin ([steps, groups, beams]
//       int32, the reordering before each step).  Writes o.bin and so.bin, shaped as q.bin and sq.bin.
#include <cstdint>
#include <fstream>
#include <iostream>
#include <string>
#include <vector>

#include "inferno/inferno.h"

using namespace Inferno;

template <typename T>
static std::vector<T> read(const std::string& path, size_t n) {
    std::vector<T> v(n);
    std::ifstream f(path, std::ios::binary);
    f.read(reinterpret_cast<char*>(v.data()), (std::streamsize)(n * sizeof(T)));
    if (!f) throw Error("cannot read " + path);
    return v;
}

static void write(const std::string& path, const std::vector<float>& v) {
    std::ofstream f(path, std::ios::binary);
    f.write(reinterpret_cast<const char*>(v.data()), (std::streamsize)(v.size() * sizeof(float)));
}

static int run(int argc, char** argv) {
    if (argc != 14) throw Error("paged_driver: 13 arguments expected");
    const std::string dir = argv[1];
    const DType dt = std::string(argv[2]) == "bf16" ? DType::BFloat16 : DType::Float32;
    size_t n[11];
    for (int i = 0; i < 11; ++i) n[i] = std::stoul(argv[3 + i]);
    const size_t G = n[0], K = n[1], L = n[2], H = n[3], D = n[4], P = n[5], S = n[6];
    const Device dev = Device::hip(0);
    PagedKVCache::Options options;
    options.page_size = n[7];
    options.beams = K;
    options.budget = n[9];
    options.recent = n[10];
    PagedKVCache cache(L, G, H, n[8], D, dev, dt, options);
    // Block i of the file's [.., rows, H, t, D] as a tensor.
    auto block = [&](const std::vector<float>& all, size_t i, size_t rows, size_t t) {
        const size_t m = rows * H * t * D;
        const std::vector<float> part(all.begin() + (std::ptrdiff_t)(i * m), all.begin() + (std::ptrdiff_t)((i + 1) * m));
        return Tensor(dt, part, std::vector<size_t>{rows, H, t, D}, "x", dev);
    };
    auto step = [&](const std::vector<float>& q, const std::vector<float>& k, const std::vector<float>& v, size_t first,
                    size_t rows, size_t t, std::vector<float>& out) {
        cache.begin(t);
        for (size_t l = 0; l < L; ++l) {
            const Tensor o = cache.attend(l, block(q, first + l, rows, t), block(k, first + l, rows, t),
                                          block(v, first + l, rows, t));
            const std::vector<float> h = o.to_host_float();
            out.insert(out.end(), h.begin(), h.end());
        }
        cache.end();
    };
    std::vector<float> o, so;
    const size_t np = L * G * H * P * D, ns = S * L * G * K * H * D;
    step(read<float>(dir + "/q.bin", np), read<float>(dir + "/k.bin", np), read<float>(dir + "/v.bin", np), 0, G, P, o);
    const std::vector<float> sq = read<float>(dir + "/sq.bin", ns), sk = read<float>(dir + "/sk.bin", ns),
                             sv = read<float>(dir + "/sv.bin", ns);
    const std::vector<int32_t> parents = K > 1 ? read<int32_t>(dir + "/parents.bin", S * G * K) : std::vector<int32_t>();
    for (size_t s = 0; s < S; ++s) {
        if (K > 1) {
            const auto at = parents.begin() + (std::ptrdiff_t)(s * G * K);
            cache.reorder(Tensor(DType::Int32, std::vector<int32_t>(at, at + (std::ptrdiff_t)(G * K)),
                                 std::vector<size_t>{G, K}, "parents", dev));
        }
        step(sq, sk, sv, s * L, G * K, 1, so);
    }
    write(dir + "/o.bin", o);
    write(dir + "/so.bin", so);
    std::cout << "length " << cache.length() << " seen " << cache.seen() << "\n";
    return 0;
}

int main(int argc, char** argv) {
    try {
        return run(argc, argv);
    } catch (const std::exception& e) {
        std::cerr << "error: " << e.what() << "\n";
        return 1;
    }
}
