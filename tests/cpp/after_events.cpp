// after_events.cpp -- foa_rx_after (include/fun_ofdm_amd.h): the next call takes the registered events with it WHATEVER it returns.  The
// library holds the caller's raw event handles; a call that was refused or failed and left them behind made a later call wait for events
// the caller had destroyed by then.  Run against hip_stub.h: no GPU, every wait is written down and a dead event's use is counted.
//
// Build / run: tests/test_host_logic.py.  Exit code 0 = all checks passed.
#include "hip_stub.h"

#include "fun_ofdm_amd.h"

#include <functional>

static int failures = 0;
#define CHECK(cond, ...) do { if (!(cond)) { failures++; printf("FAIL line %d: ", __LINE__); printf(__VA_ARGS__); printf("\n"); } } while (0)

static const size_t kN = 4000, kSlot = 64;
static std::vector<float> iq(2 * kN), iq_out(2 * kN);
static std::vector<double> iq64(2 * kN), frames(2 * kN);
static std::vector<foa_frame_desc> descs(16);
static std::vector<int64_t> ends(16, kN);
static std::vector<uint8_t> psdu(16 * kSlot), pay(256);
static std::vector<foa_frame_result> res(16);

static int decode(foa_rx *rx) { return foa_rx_decode_frames_dev(rx, iq.data(), kN, descs.data(), ends.data(), 2, psdu.data(), kSlot, res.data()); }

// waits for any of ev among the operations queued since the last look; *ahead: all of them in front of the first copy, fill or launch
static int waits_for(const std::vector<hipEvent_t> &ev, bool *ahead = nullptr)
{
    int n = 0;
    bool work = false;
    if (ahead) *ahead = true;
    for (const stub::Op &o : stub::taken()) {
        if (o.what == "copy" || o.what == "fill" || o.what == "launch") work = true;
        if (o.what != "wait") continue;
        for (hipEvent_t e : ev) if (o.event == e) { n++; if (ahead && work) *ahead = false; }
    }
    return n;
}

// registers `n` events, makes the call, destroys the events, then decodes: nothing may wait for them any more
static void leaves_nothing(const char *what, bool ok_wanted, const std::function<int(foa_rx *, hipEvent_t)> &call, int n = 2)
{
    foa_rx *rx = nullptr;
    if (foa_rx_create(&rx, 0)) { CHECK(false, "%s: foa_rx_create: %s", what, foa_last_error()); return; }
    std::vector<hipEvent_t> ev(n);
    for (auto &e : ev) { (void)hipEventCreate(&e); CHECK(foa_rx_after(rx, e) == FOA_OK, "%s: foa_rx_after", what); }
    hipEvent_t one_more;
    (void)hipEventCreate(&one_more);
    const int rc = call(rx, one_more);
    stub::fail_malloc = stub::fail_set_device = false;
    CHECK((rc == FOA_OK) == ok_wanted, "%s: returned %d (%s)", what, rc, foa_last_error());
    ev.push_back(one_more);
    for (auto e : ev) (void)hipEventDestroy(e);
    stub::taken();
    stub::dead_event_uses = 0;
    CHECK(decode(rx) == FOA_OK, "%s: the next call: %s", what, foa_last_error());
    CHECK(waits_for(ev) == 0 && stub::dead_event_uses == 0, "%s: the next call waits for the caller's destroyed events (%d uses)", what, stub::dead_event_uses);
    foa_rx_destroy(rx);
}

// ... and a call that does queue work waits for each of them once, in front of everything else it queues
static void waits_once(const char *what, const std::function<int(foa_rx *)> &call)
{
    foa_rx *rx = nullptr;
    if (foa_rx_create(&rx, 0)) { CHECK(false, "%s: foa_rx_create: %s", what, foa_last_error()); return; }
    std::vector<hipEvent_t> ev(16);
    for (auto &e : ev) { (void)hipEventCreate(&e); CHECK(foa_rx_after(rx, e) == FOA_OK, "%s: foa_rx_after", what); }
    stub::taken();
    CHECK(call(rx) == FOA_OK, "%s: %s", what, foa_last_error());
    bool ahead = false;
    const int n = waits_for(ev, &ahead);
    CHECK(n == 16 && ahead, "%s: %d waits for 16 events%s", what, n, ahead ? "" : ", some behind the first work");
    for (auto e : ev) (void)hipEventDestroy(e);
    stub::dead_event_uses = 0;
    CHECK(decode(rx) == FOA_OK && waits_for(ev) == 0 && stub::dead_event_uses == 0, "%s: the call after it waits again", what);
    foa_rx_destroy(rx);
}

int main()
{
    const float *q = iq.data();
    foa_frame_desc *d = descs.data();
    int64_t *e = ends.data();
    uint8_t *p = psdu.data();
    foa_frame_result *r = res.data();
    size_t n = 0;
    uint64_t t = 0;
    for (size_t i = 0; i < descs.size(); i++) descs[i] = { (int64_t)(200 * i), 0, 1, 0, 1, 0 };

    // the batch decode call
    leaves_nothing("decode, NULL samples", false, [&](foa_rx *rx, hipEvent_t) { return foa_rx_decode_frames_dev(rx, nullptr, kN, d, e, 2, p, kSlot, r); });
    leaves_nothing("decode, too many frames", false, [&](foa_rx *rx, hipEvent_t) { return foa_rx_decode_frames_dev(rx, q, kN, d, e, (size_t)1 << 40, p, kSlot, r); });
    leaves_nothing("decode, too much context", false, [&](foa_rx *rx, hipEvent_t) { return foa_rx_decode_frames_ctx_dev(rx, q, kN, d, e, 2, (size_t)1 << 40, p, kSlot, r); });
    leaves_nothing("decode, no frames", true, [&](foa_rx *rx, hipEvent_t) { return foa_rx_decode_frames_dev(rx, q, kN, d, e, 0, p, kSlot, r); });
    leaves_nothing("decode, too many in front", false, [&](foa_rx *rx, hipEvent_t) { return foa_rx_decode_frames_lead_ctx_dev(rx, q, kN, d, e, (size_t)1 << 40, 2, 0, p, kSlot, r); });
    leaves_nothing("decode, NULL descriptors", false, [&](foa_rx *rx, hipEvent_t) { return foa_rx_decode_frames_lead_ctx_dev(rx, q, kN, nullptr, e, 1, 2, 0, p, kSlot, r); });
    leaves_nothing("decode, no device", false, [&](foa_rx *rx, hipEvent_t) { stub::fail_set_device = true; return decode(rx); });
    leaves_nothing("decode, no memory", false, [&](foa_rx *rx, hipEvent_t) { stub::fail_malloc = true; return decode(rx); });
    leaves_nothing("decode _after, NULL samples", false, [&](foa_rx *rx, hipEvent_t x) { return foa_rx_decode_frames_dev_after(rx, x, nullptr, kN, d, e, 2, p, kSlot, r); });
    leaves_nothing("decode _after, one event too many", false, [&](foa_rx *rx, hipEvent_t x) { return foa_rx_decode_frames_dev_after(rx, x, q, kN, d, e, 2, p, kSlot, r); }, 16);

    // its host-pointer forms
    leaves_nothing("decode_host, NULL", false, [&](foa_rx *rx, hipEvent_t) { return foa_rx_decode_frames_host(rx, nullptr, kN, d, e, 2, p, kSlot, r); });
    leaves_nothing("decode_host, no frames", true, [&](foa_rx *rx, hipEvent_t) { return foa_rx_decode_frames_host(rx, q, kN, d, e, 0, p, kSlot, r); });
    leaves_nothing("decode_host, no memory", false, [&](foa_rx *rx, hipEvent_t) { stub::fail_malloc = true; return foa_rx_decode_frames_host(rx, q, kN, d, e, 2, p, kSlot, r); });
    leaves_nothing("decode_f64_host, NULL", false, [&](foa_rx *rx, hipEvent_t) { return foa_rx_decode_frames_f64_host(rx, iq64.data(), kN, d, nullptr, 2, p, kSlot, r); });
    leaves_nothing("submit_host, NULL ticket", false, [&](foa_rx *rx, hipEvent_t) { return foa_rx_submit_host(rx, q, kN, d, e, 2, kSlot, nullptr); });
    leaves_nothing("submit_host, no frames", false, [&](foa_rx *rx, hipEvent_t) { return foa_rx_submit_host(rx, q, kN, d, e, 0, kSlot, &t); });
    leaves_nothing("submit_host, no memory", false, [&](foa_rx *rx, hipEvent_t) { stub::fail_malloc = true; return foa_rx_submit_host(rx, q, kN, d, e, 2, kSlot, &t); });
    leaves_nothing("submit_host, eight in flight", false, [&](foa_rx *rx, hipEvent_t x) {
        for (int i = 0; i < 8; i++) if (foa_rx_submit_host(rx, q, kN, d, e, 2, kSlot, &t)) return (int)FOA_OK;
        (void)foa_rx_after(rx, x);
        return foa_rx_submit_host(rx, q, kN, d, e, 2, kSlot, &t); });

    // the pre-sync
    leaves_nothing("sync_dev_begin, NULL", false, [&](foa_rx *rx, hipEvent_t) { return foa_rx_sync_dev_begin(rx, q, kN, nullptr, e, 16); });
    leaves_nothing("sync_dev_begin, too long", false, [&](foa_rx *rx, hipEvent_t) { return foa_rx_sync_dev_begin(rx, q, (size_t)1 << 40, d, e, 16); });
    leaves_nothing("sync_dev_begin, no samples", true, [&](foa_rx *rx, hipEvent_t) { return foa_rx_sync_dev_begin(rx, q, 0, d, e, 16); });
    leaves_nothing("sync_dev_begin, in flight already", false, [&](foa_rx *rx, hipEvent_t x) {
        if (foa_rx_sync_dev_begin(rx, q, kN, d, e, 16)) return (int)FOA_OK;
        (void)foa_rx_after(rx, x);
        return foa_rx_sync_dev_begin(rx, q, kN, d, e, 16); });
    leaves_nothing("sync_dev_begin, no memory", false, [&](foa_rx *rx, hipEvent_t) { stub::fail_malloc = true; return foa_rx_sync_dev_begin(rx, q, kN, d, e, 16); });
    leaves_nothing("sync_dev, NULL count", false, [&](foa_rx *rx, hipEvent_t) { return foa_rx_sync_dev(rx, q, kN, d, e, 16, nullptr); });
    leaves_nothing("sync_dev_begin _after, NULL", false, [&](foa_rx *rx, hipEvent_t x) { return foa_rx_sync_dev_begin_after(rx, x, nullptr, kN, d, e, 16); });
    leaves_nothing("sync_dev_begin _after, one event too many", false, [&](foa_rx *rx, hipEvent_t x) { return foa_rx_sync_dev_begin_after(rx, x, q, kN, d, e, 16); }, 16);

    // the transmit side
    leaves_nothing("build_frames, bad rate", false, [&](foa_rx *rx, hipEvent_t) { return foa_tx_build_frames_dev(rx, pay.data(), 10, 10, 99, 1, frames.data(), &n); });
    leaves_nothing("build_frames, NULL", false, [&](foa_rx *rx, hipEvent_t) { return foa_tx_build_frames_dev(rx, nullptr, 10, 10, 10, 1, frames.data(), &n); });
    leaves_nothing("build_frames, NULL size", false, [&](foa_rx *rx, hipEvent_t) { return foa_tx_build_frames_dev(rx, pay.data(), 10, 10, 10, 1, frames.data(), nullptr); });
    leaves_nothing("build_frames, short pitch", false, [&](foa_rx *rx, hipEvent_t) { return foa_tx_build_frames_dev(rx, pay.data(), 9, 10, 10, 2, frames.data(), &n); });
    leaves_nothing("build_frames, no memory", false, [&](foa_rx *rx, hipEvent_t) { stub::fail_malloc = true; return foa_tx_build_frames_dev(rx, pay.data(), 10, 10, 10, 1, frames.data(), &n); });
    leaves_nothing("channel, no frames", true, [&](foa_rx *rx, hipEvent_t) { return foa_tx_channel_dev(rx, frames.data(), 0, 480, 600, 10, 25, 0, 1, iq_out.data()); });
    leaves_nothing("channel, NULL", false, [&](foa_rx *rx, hipEvent_t) { return foa_tx_channel_dev(rx, frames.data(), 1, 480, 600, 10, 25, 0, 1, nullptr); });
    leaves_nothing("channel, short pitch", false, [&](foa_rx *rx, hipEvent_t) { return foa_tx_channel_dev(rx, frames.data(), 1, 480, 400, 10, 25, 0, 1, iq_out.data()); });

    // a stream engine: it reads no device memory of the caller's, and its submitter thread must not find the events later
    leaves_nothing("stream_create, bad batch", false, [&](foa_rx *rx, hipEvent_t) { foa_stream *s = nullptr; return foa_stream_create(rx, 100, 0, &s); });
    leaves_nothing("stream_create", true, [&](foa_rx *rx, hipEvent_t) {
        foa_stream *s = nullptr;
        const int rc = foa_stream_create(rx, 4096, 0, &s);
        if (!rc) foa_stream_destroy(s);
        return rc; });

    waits_once("decode", decode);
    waits_once("decode in line", [](foa_rx *rx) { const int rc = foa_rx_set_option(rx, "pipeline", 0); return rc ? rc : decode(rx); });
    waits_once("decode_host", [&](foa_rx *rx) { return foa_rx_decode_frames_host(rx, q, kN, d, e, 2, p, kSlot, r); });
    waits_once("submit_host", [&](foa_rx *rx) { return foa_rx_submit_host(rx, q, kN, d, e, 2, kSlot, &t); });
    waits_once("sync_dev_begin", [&](foa_rx *rx) { return foa_rx_sync_dev_begin(rx, q, kN, d, e, 16); });
    waits_once("build_frames", [&](foa_rx *rx) { return foa_tx_build_frames_dev(rx, pay.data(), 10, 10, 10, 1, frames.data(), &n); });
    // (asking for a frame's size queues nothing and takes nothing: the call that builds the frames still waits)
    waits_once("build_frames behind the size query", [&](foa_rx *rx) {
        const int rc = foa_tx_build_frames_dev(rx, nullptr, 0, 10, 10, 0, nullptr, &n);
        return rc ? rc : foa_tx_build_frames_dev(rx, pay.data(), 10, 10, 10, 1, frames.data(), &n); });
    waits_once("channel", [&](foa_rx *rx) { return foa_tx_channel_dev(rx, frames.data(), 1, 480, 600, 10, 25, 0, 1, iq_out.data()); });

    // too many events for one call are refused, the sixteen stay for the call
    {
        foa_rx *rx = nullptr;
        CHECK(foa_rx_create(&rx, 0) == FOA_OK, "%s", foa_last_error());
        std::vector<hipEvent_t> ev(17);
        for (auto &x : ev) (void)hipEventCreate(&x);
        for (int i = 0; i < 16; i++) CHECK(foa_rx_after(rx, ev[i]) == FOA_OK, "event %d", i);
        CHECK(foa_rx_after(rx, ev[16]) == FOA_E_STATE && foa_rx_after(rx, nullptr) == FOA_E_INVALID, "the 17th event");
        stub::taken();
        CHECK(decode(rx) == FOA_OK && waits_for(ev) == 16, "the sixteen events");
        foa_rx_destroy(rx);
    }
    printf("%s\n", failures ? "FAILED" : "after_events: all checks passed");
    return failures ? 1 : 0;
}
