// Workspaces of calls that may be made on several streams, from several threads and into several CUDA graphs (host code).
//
//   one stream       the first stream that asks keeps a workspace of its own; nothing is recorded or waited for.
//   further streams  share a few more, each with an event behind its last use that the next stream to take it waits for.
//   a captured call  takes a workspace that belongs to its graph (and to its stream in it), so graphs replay side by side.  The
//                    graph holds a user object; when it and what was instantiated from it are gone, the next capture takes over.
//   growing          allocates anew and keeps the old allocation until the context goes: nothing is synchronised, calls in
//                    flight and captured graphs keep their addresses, and a capture may grow too.
//
// A pick, the launches on what was picked and done() go together under `mu`.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <memory>
#include <mutex>
#include <new>
#include <vector>

namespace lq4 {

enum ScratchKind { kScratchAttend, kScratchVerify, kScratchKinds };

struct Scratch {
    void* p[kScratchKinds] = {};
    size_t cap[kScratchKinds] = {};
    cudaEvent_t used = nullptr;               // further streams: behind the last use
    unsigned long long stream = 0, capture = 0;
    uint64_t turn = 0;
    std::shared_ptr<std::atomic<bool>> live;  // graphs: false once the graph is gone
};

class ScratchPool {
  public:
    std::mutex mu;

    // The workspace for a call on `s`, on the current device.  may_grow false: only what there is, which the first
    // stream's calls use too.
    cudaError_t pick(cudaStream_t s, bool may_grow, Scratch** out) try {
        cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
        unsigned long long capture = 0, id = 0;
        cudaGraph_t graph = nullptr;
        cudaError_t e = cudaStreamGetCaptureInfo(s, &status, &capture, &graph);
        if (e != cudaSuccess) return e;
        if (status == cudaStreamCaptureStatusInvalidated) return cudaErrorStreamCaptureInvalidated;
        // (a stream that captures has no id to ask for, but its handle is its own until the capture ends)
        const bool capturing = status == cudaStreamCaptureStatusActive;
        if (capturing && may_grow) return pick_graph(graph, capture, reinterpret_cast<uintptr_t>(s), out);
        if (!capturing && (e = cudaStreamGetId(s, &id)) != cudaSuccess) return e;
        if (streams_.empty()) {
            streams_.push_back(std::unique_ptr<Scratch>(new Scratch));
            streams_[0]->stream = id;
        }
        Scratch* w = may_grow ? nullptr : streams_[0].get();
        for (auto& x : streams_)
            if (x->stream == id) w = x.get();
        if (!w) {
            if (streams_.size() < kMaxStreams) {
                std::unique_ptr<Scratch> x(new Scratch);
                if ((e = cudaEventCreateWithFlags(&x->used, cudaEventDisableTiming)) != cudaSuccess) return e;
                streams_.push_back(std::move(x));
                w = streams_.back().get();
            } else {
                w = streams_[1].get();
                for (size_t i = 2; i < streams_.size(); ++i)
                    if (streams_[i]->turn < w->turn) w = streams_[i].get();
                if ((e = cudaStreamWaitEvent(s, w->used, 0)) != cudaSuccess) return e;
            }
            w->stream = id;
        }
        w->turn = ++turn_;
        *out = w;
        return cudaSuccess;
    } catch (const std::bad_alloc&) {
        return cudaErrorMemoryAllocation;
    }

    // At least `bytes` of `kind`.
    cudaError_t grow(Scratch& w, ScratchKind kind, size_t bytes) try {
        if (bytes <= w.cap[kind]) return cudaSuccess;
        outgrown_.reserve(outgrown_.size() + 1);
        Relaxed guard;
        void* p = nullptr;
        const size_t cap = (bytes + 255) / 256 * 256;
        const cudaError_t e = cudaMalloc(&p, cap);
        if (e != cudaSuccess) {
            cudaGetLastError();
            return e;
        }
        if (w.p[kind]) outgrown_.push_back(w.p[kind]);
        w.p[kind] = p;
        w.cap[kind] = cap;
        return cudaSuccess;
    } catch (const std::bad_alloc&) {
        return cudaErrorMemoryAllocation;
    }

    // Behind the launches of a call.
    cudaError_t done(Scratch& w, cudaStream_t s) { return w.used ? cudaEventRecord(w.used, s) : cudaSuccess; }

    void free_all() {
        for (auto* list : {&streams_, &graphs_}) {
            for (auto& x : *list) {
                for (void* p : x->p)
                    if (p) cudaFree(p);
                if (x->used) cudaEventDestroy(x->used);
            }
            list->clear();
        }
        for (void* p : outgrown_) cudaFree(p);
        outgrown_.clear();
    }

  private:
    static constexpr size_t kMaxStreams = 5;

    // An allocation disturbs no capture, neither this thread's nor another one's.
    struct Relaxed {
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        Relaxed() { cudaThreadExchangeStreamCaptureMode(&mode); }
        ~Relaxed() { cudaThreadExchangeStreamCaptureMode(&mode); }
    };

    cudaError_t pick_graph(cudaGraph_t graph, unsigned long long capture, unsigned long long id, Scratch** out) {
        Scratch* w = nullptr;
        for (auto& x : graphs_) {
            if (!x->live->load(std::memory_order_acquire)) {
                if (!w || x->cap[kScratchAttend] > w->cap[kScratchAttend]) w = x.get();
            } else if (x->capture == capture && x->stream == id) {
                *out = x.get();
                return cudaSuccess;
            }
        }
        Relaxed guard;
        typedef std::shared_ptr<std::atomic<bool>> Flag;
        Flag live = std::make_shared<std::atomic<bool>>(true);
        if (!w) {
            std::unique_ptr<Scratch> x(new Scratch);
            x->live = std::make_shared<std::atomic<bool>>(false);
            graphs_.push_back(std::move(x));
            w = graphs_.back().get();
        }
        std::unique_ptr<Flag> held(new Flag(live));
        cudaUserObject_t object = nullptr;
        auto gone = [](void* at) {
            std::unique_ptr<Flag> flag(static_cast<Flag*>(at));
            (*flag)->store(false, std::memory_order_release);
        };
        cudaError_t e = cudaUserObjectCreate(&object, held.get(), gone, 1, cudaUserObjectNoDestructorSync);
        if (e != cudaSuccess) return e;
        held.release();
        if ((e = cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove)) != cudaSuccess) {
            cudaUserObjectRelease(object, 1);
            return e;
        }
        w->live = live;
        w->capture = capture;
        w->stream = id;
        *out = w;
        return cudaSuccess;
    }

    std::vector<std::unique_ptr<Scratch>> streams_, graphs_;
    std::vector<void*> outgrown_;
    uint64_t turn_ = 0;
};

}  // namespace lq4
