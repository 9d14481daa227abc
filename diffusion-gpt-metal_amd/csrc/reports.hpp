// Words in which kernels report to their context what they find wrong in data that only
// the device reads. Plain C++, so that it also runs on the host.
#pragma once
#include <cstdint>
#include <mutex>

namespace dgm {

// Four words a context, from blocks of host memory that the device writes. None is handed out
// twice, nor freed: a captured graph may outlive the context that it reports to, and then
// writes where nobody reads. That is 16 bytes for each context of a process.
class ReportWords {
public:
    static constexpr int kWords = 4, kContexts = 512;   // of a context; contexts of a block
    // alloc(bytes): such memory, or nullptr, which is then the result.
    template <typename Alloc>
    uint32_t* take(const Alloc& alloc) {
        std::lock_guard<std::mutex> lock(mu_);
        if (left_ == 0) {
            next_ = static_cast<uint32_t*>(alloc(kContexts * kWords * sizeof(uint32_t)));
            if (!next_) return nullptr;
            left_ = kContexts;
        }
        uint32_t* const words = next_;
        next_ += kWords;
        --left_;
        for (int i = 0; i < kWords; ++i) words[i] = 0;
        return words;
    }

private:
    std::mutex mu_;
    uint32_t* next_ = nullptr;
    int left_ = 0;
};

}  // namespace dgm
