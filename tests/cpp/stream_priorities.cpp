// stream_priorities.cpp -- every HIP stream of the library is made at the default priority: work on streams of different priorities side by
// side has hung GPUs this library runs on, for good.  Handles, a stream engine, a shard engine and the stream that joins the others for a
// caller's event are made against hip_stub.h (no GPU), which writes down every stream's priority.
//
// Build / run: tests/test_host_logic.py.  Exit code 0 = all checks passed.
#include "hip_stub.h"

#include "fun_ofdm_amd.h"

static int failures = 0;
#define CHECK(cond, ...) do { if (!(cond)) { failures++; printf("FAIL line %d: ", __LINE__); printf(__VA_ARGS__); printf("\n"); } } while (0)

static size_t seen = 0;
static void all_default(const char *what, size_t at_least)
{
    CHECK(stub::streams.size() >= seen + at_least, "%s: %zu streams made", what, stub::streams.size() - seen);
    for (size_t i = seen; i < stub::streams.size(); i++) {
        CHECK(stub::streams[i]->priority == 0, "%s: stream %zu at priority %d", what, i - seen, stub::streams[i]->priority);
        CHECK(stub::streams[i]->flags == hipStreamNonBlocking, "%s: stream %zu with flags %u", what, i - seen, stub::streams[i]->flags);
    }
    seen = stub::streams.size();
}

int main()
{
    foa_rx *rx = nullptr;
    CHECK(foa_rx_create(&rx, 0) == FOA_OK, "%s", foa_last_error());
    all_default("foa_rx_create", 6);
    hipEvent_t e;
    (void)hipEventCreate(&e);
    CHECK(foa_rx_record_consumed(rx, e) == FOA_OK && foa_rx_record_done(rx, e) == FOA_OK, "%s", foa_last_error());
    all_default("foa_rx_record_consumed / _done", 1);
    for (size_t batch : { (size_t)4096, (size_t)1 << 17 }) {
        foa_stream *s = nullptr;
        CHECK(foa_stream_create(rx, batch, 0, &s) == FOA_OK, "%s", foa_last_error());
        all_default("foa_stream_create", 1);
        foa_stream_destroy(s);
    }
    foa_rx_destroy(rx);
    const int devices[2] = { 0, 0 };
    foa_shard *sh = nullptr;
    CHECK(foa_shard_create(devices, 2, 1 << 17, 0, &sh) == FOA_OK, "%s", foa_last_error());
    all_default("foa_shard_create", 2 * (6 + 2));
    foa_shard_destroy(sh);
    printf("%s\n", failures ? "FAILED" : "stream_priorities: all checks passed");
    return failures ? 1 : 0;
}
