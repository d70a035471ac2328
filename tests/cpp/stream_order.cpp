// stream_order.cpp -- a handle's streams sit on hardware queues that do not get in each other's way, whatever streams the host has made before.
// The runtime gives a new stream a queue of its own while its pool of four is not full, and the least used queue after that (of several, the
// first in an order of its own).  That rule is played here over the streams the library makes against hip_stub.h (no GPU), for every such
// order and for hosts of 0 .. 6 streams; which stream does what is read off what is queued on it.
//
// Build / run: tests/test_host_logic.py.  Exit code 0 = all checks passed.
#include "hip_stub.h"

#include <algorithm>
#include <set>

#include "fun_ofdm_amd.h"

static int failures = 0;
#define CHECK(cond, ...) do { if (!(cond)) { failures++; printf("FAIL line %d: ", __LINE__); printf(__VA_ARGS__); printf("\n"); } } while (0)

static const size_t n = 4000, slot = 64;
static std::vector<float> iq(2 * n);
static std::vector<foa_frame_desc> descs(2, { 0, 0, 1, 0, 1, 0 });
static std::vector<int64_t> ends(2, (int64_t)n);
static std::vector<uint8_t> psdu(2 * slot);
static std::vector<foa_frame_result> res(2);

static const void *launched(const std::vector<stub::Op> &ops, const char *kernel)
{
    for (const stub::Op &o : ops) if (o.what == "launch" && o.name.find(kernel) != std::string::npos) return o.stream;
    return nullptr;
}
static std::vector<stub::Op> decode(foa_rx *rx)
{
    CHECK(foa_rx_decode_frames_dev(rx, iq.data(), n, descs.data(), ends.data(), 2, psdu.data(), slot, res.data()) == FOA_OK, "%s", foa_last_error());
    return stub::taken();
}

int main()
{
    for (int host = 0; host <= 6; host++) {
        const size_t first = stub::streams.size();
        for (int i = 0; i < host; i++) { hipStream_t s; (void)hipStreamCreate(&s); }
        foa_rx *rx = nullptr;
        CHECK(foa_rx_create(&rx, 0) == FOA_OK, "%s", foa_last_error());
        const std::vector<stub::Stream *> made(stub::streams.begin() + first, stub::streams.end());
        stub::taken();
        // which stream is which
        CHECK(foa_rx_decode_frames_host(rx, iq.data(), n, descs.data(), ends.data(), 2, psdu.data(), slot, res.data()) == FOA_OK, "%s", foa_last_error());
        const std::vector<stub::Op> lone = stub::taken();
        const void *copies = nullptr, *stitch = launched(lone, "k_tb_finish"), *lane[4];
        for (const stub::Op &o : lone) if (o.what == "copy" && !copies) copies = o.stream;
        CHECK(foa_rx_sync(rx) == FOA_OK && foa_rx_set_option(rx, "depth", 4) == FOA_OK, "%s", foa_last_error());
        lane[0] = launched(lone, "k_header");                  // the first call since the handle was made
        for (int k = 1; k < 4; k++) lane[k] = launched(decode(rx), "k_header");
        const std::set<const void *> all = { copies, stitch, lane[0], lane[1], lane[2], lane[3] };
        CHECK(all.size() == 6 && !all.count(nullptr), "six streams of their own: copies %p stitch %p lanes %p %p %p %p", copies, stitch, lane[0], lane[1], lane[2], lane[3]);
        if (failures) break;
        // how many loops a call keeps in flight when it is left to the library: three; two where a pre-sync or copies run on the copy stream
        CHECK(foa_rx_set_option(rx, "depth", 0) == FOA_OK, "%s", foa_last_error());
        std::set<const void *> used;
        for (int k = 0; k < 6; k++) used.insert(launched(decode(rx), "k_header"));
        CHECK((used == std::set<const void *>{ lane[0], lane[1], lane[2] }), "small calls: %zu lanes", used.size());
        used.clear();
        for (int k = 0; k < 6; k++) {
            std::vector<foa_frame_desc> d(64);
            std::vector<int64_t> e(64);
            size_t got = 0;
            CHECK(foa_rx_sync_dev(rx, iq.data(), n, d.data(), e.data(), 64, &got) == FOA_OK, "%s", foa_last_error());
            stub::taken();
            used.insert(launched(decode(rx), "k_header"));
        }
        CHECK((used == std::set<const void *>{ lane[0], lane[1] }), "small calls behind a pre-sync: %zu lanes", used.size());
        // the queues
        int pi[4] = { 0, 1, 2, 3 };
        do {
            int count[4] = { 0, 0, 0, 0 };
            size_t queues = 0;
            std::map<const void *, int> q;
            for (stub::Stream *s : made) {
                int k = 0;
                if (queues < 4) k = (int)queues++;
                else {
                    k = pi[0];
                    for (int i = 1; i < 4; i++) if (count[pi[i]] < count[k]) k = pi[i];
                }
                count[k]++;
                q[s] = k;
            }
            auto apart = [&](std::vector<const void *> s) { std::set<int> on; for (const void *x : s) on.insert(q.at(x)); return on.size() == s.size(); };
            CHECK(apart({ lane[0], lane[1], stitch, copies }), "host %d, order %d%d%d%d: a machine-filling call's streams share a queue", host, pi[0], pi[1], pi[2], pi[3]);
            CHECK(apart({ lane[0], lane[1], lane[2], stitch }), "host %d, order %d%d%d%d: three lanes and the stitch stream share a queue", host, pi[0], pi[1], pi[2], pi[3]);
            CHECK(apart({ lane[0], lane[1], lane[2], lane[3] }), "host %d, order %d%d%d%d: four lanes share a queue", host, pi[0], pi[1], pi[2], pi[3]);
        } while (std::next_permutation(pi, pi + 4) && failures < 20);
        foa_rx_destroy(rx);
    }
    printf("%s\n", failures ? "FAILED" : "stream_order: all checks passed");
    return failures ? 1 : 0;
}
