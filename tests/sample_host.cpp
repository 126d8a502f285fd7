// The drawing kernels on the host (host_gpu/hip/hip_runtime.h), as a library for the tests.
#include "../telmo_amd/csrc/kernels_sample.hip"

extern "C" int draw_on_host(uint32_t type, const void *logits, long ld, int rows, int n, float temperature, int top_k, float top_p,
                            float min_p, const float *uniforms, int32_t *tokens, float *probs, int first_wave) {
    std::vector<uint64_t> work(tg::sample_work_bytes(rows, n) / 8 + 1, 0xa5a5a5a5a5a5a5a5ull);
    const tg::SampleArgs a{logits, ld, n, temperature, top_p, min_p, top_k, nullptr, nullptr, nullptr, nullptr, uniforms, tokens, probs};
    host_gpu::first_wave = first_wave;
    host_gpu::all_finished = true;
    const hipError_t e = tg::launch_sample(a, type, rows, work.data(), nullptr);
    return e == hipSuccess && host_gpu::all_finished ? 0 : 1;
}
