// scratch_order.cpp -- foa_tx_build_frames_dev returns while its kernels still read the handle's staging buffer on the handle's first stream;
// the host-pointer decode calls copy their inputs into the SAME buffer on another stream.  Those copies must be behind the frames: checked on
// the order of what is queued, against hip_stub.h (no GPU).
//
// Build / run: tests/test_host_logic.py.  Exit code 0 = all checks passed.
#include "hip_stub.h"

#include "fun_ofdm_amd.h"

static int failures = 0;
#define CHECK(cond, ...) do { if (!(cond)) { failures++; printf("FAIL line %d: ", __LINE__); printf(__VA_ARGS__); printf("\n"); } } while (0)

int main()
{
    const size_t n = 4000, slot = 64;
    std::vector<float> iq(2 * n);
    std::vector<double> iq64(2 * n), frames(16 * n);
    std::vector<foa_frame_desc> descs(2, { 0, 0, 1, 0, 1, 0 });
    std::vector<int64_t> ends(2, (int64_t)n);
    std::vector<uint8_t> psdu(2 * slot), pay(4096);
    std::vector<foa_frame_result> res(2);
    for (int pipeline = 0; pipeline < 2; pipeline++)
        for (int f64 = 0; f64 < 2; f64++)
            for (int calls = 1; calls <= 2; calls++) {
                foa_rx *rx = nullptr;
                size_t fs = 0;
                CHECK(foa_rx_create(&rx, 0) == FOA_OK && foa_rx_set_option(rx, "pipeline", pipeline) == FOA_OK, "%s", foa_last_error());
                auto decode = [&] {
                    return f64 ? foa_rx_decode_frames_f64_host(rx, iq64.data(), n, descs.data(), ends.data(), 2, psdu.data(), slot, res.data())
                               : foa_rx_decode_frames_host(rx, iq.data(), n, descs.data(), ends.data(), 2, psdu.data(), slot, res.data());
                };
                CHECK(decode() == FOA_OK, "%s", foa_last_error());            // (the staging buffer has its size: the next call frees nothing, which would wait)
                stub::taken();
                for (int k = 0; k < calls; k++) CHECK(foa_tx_build_frames_dev(rx, pay.data(), 100, 100, 10, 4, frames.data(), &fs) == FOA_OK, "%s", foa_last_error());
                const void *tx_stream = nullptr, *tx_event = nullptr;         // where the last frames' kernels are, and the last event behind them
                for (const stub::Op &o : stub::taken()) {
                    if (o.what == "launch" && o.name.find("k_tx_") != std::string::npos) { tx_stream = o.stream; tx_event = nullptr; }
                    if (o.what == "record" && o.stream == tx_stream) tx_event = o.event;
                }
                CHECK(tx_stream, "no transmit kernel was launched");
                CHECK(decode() == FOA_OK, "%s", foa_last_error());
                const void *copy_stream = nullptr;
                bool waited = false;
                for (const stub::Op &o : stub::taken()) {
                    if (o.what == "wait" && o.event == tx_event && tx_event) { waited = true; copy_stream = o.stream; }
                    if (o.what == "copy" || o.what == "fill") {
                        CHECK(o.stream == tx_stream || (waited && o.stream == copy_stream), "pipeline %d, f64 %d, %d calls: the staging copy is not behind the frames", pipeline, f64, calls);
                        break;
                    }
                }
                foa_rx_destroy(rx);
            }
    printf("%s\n", failures ? "FAILED" : "scratch_order: all checks passed");
    return failures ? 1 : 0;
}
