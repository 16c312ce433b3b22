// verify_threads.cpp -- gbx_verify_tokens from two host threads at once, on streams
// of their own, with sizes that need very different amounts of shared memory.
// Every call has to be launched, and the last one's tokens to be the greedy ones
// (temperature 1 over one-hot rows).  Prints "ok", or what was refused.
#include <cstdio>
#include <cstdlib>
#include <string>
#include <thread>
#include <vector>

#include <cuda_runtime.h>

#include "gbx.h"

static std::string run(int calls, int n, int vocab)
{
    const int rows = n + 1;
    std::vector<float> logits((size_t)rows * vocab, 0.0f);
    std::vector<int32_t> ids(n + 1), out(rows, -9);
    std::vector<double> u(rows, 0.25);
    for (int i = 0; i < rows; ++i) {
        ids[i] = (7 * i + 3) % vocab;
        logits[(size_t)i * vocab + ids[i]] = 200.0f;   // all of the probability
    }
    float* dl;
    double* du;
    int32_t *di, *dout, *dacc;
    cudaStream_t st;
    if (cudaMalloc(&dl, logits.size() * 4) || cudaMalloc(&du, rows * 8) || cudaMalloc(&di, rows * 4) || cudaMalloc(&dout, rows * 4) ||
        cudaMalloc(&dacc, 4) || cudaStreamCreateWithFlags(&st, cudaStreamNonBlocking) ||
        cudaMemcpy(dl, logits.data(), logits.size() * 4, cudaMemcpyHostToDevice) ||
        cudaMemcpy(du, u.data(), rows * 8, cudaMemcpyHostToDevice) || cudaMemcpy(di, ids.data(), rows * 4, cudaMemcpyHostToDevice))
        return "setting up failed";
    for (int c = 0; c < calls; ++c)
        if (gbx_verify_tokens(dl, nullptr, di, nullptr, 1, n, vocab, 1.0, du, dout, dacc, nullptr, reinterpret_cast<gbx_stream_t>(st)))
            return std::string("call refused: ") + gbx_last_error();
    int32_t acc = -9;
    if (cudaStreamSynchronize(st) || cudaMemcpy(out.data(), dout, rows * 4, cudaMemcpyDeviceToHost) ||
        cudaMemcpy(&acc, dacc, 4, cudaMemcpyDeviceToHost))
        return "reading back failed";
    return acc == n && out == ids ? "" : "wrong tokens";
}

int main(int, char** argv)
{
    const int calls = std::atoi(argv[1]);
    std::string a, b;
    std::thread first([&] { a = run(calls, 100, 64); }), second([&] { b = run(calls, 1, 64); });
    first.join();
    second.join();
    if (!a.empty() || !b.empty()) {
        std::printf("%s | %s\n", a.c_str(), b.c_str());
        return 1;
    }
    std::printf("ok\n");
    return 0;
}
