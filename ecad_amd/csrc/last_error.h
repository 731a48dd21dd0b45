// last_error.h -- the message of a failed call, kept for ecad_last_error.  Calls of several threads on one engine may fail at once: each thread finds the message of its own
// last failure, and one that had none here the engine's last.
#pragma once
#include <atomic>
#include <cstdint>
#include <mutex>
#include <string>

namespace ecad {

class LastError {
 public:
  LastError() : id_(next()) {}
  LastError(const LastError&) = delete;
  LastError& operator=(const LastError&) = delete;

  void set(const char* text) noexcept {
    try {
      Mine& m = mine();
      m.of = 0;  // (no half a message where memory runs out)
      m.text = text;
      std::lock_guard<std::mutex> hold(lock_);
      last_ = text;
      m.of = id_;
    } catch (...) {
    }
  }
  // good until this thread's next failure or question
  const char* get() const noexcept {
    try {
      Mine& m = mine();
      if (m.of == id_) return m.text.c_str();
      std::lock_guard<std::mutex> hold(lock_);
      m.other = last_;
      return m.other.c_str();
    } catch (...) {
      return "";
    }
  }

 private:
  struct Mine {
    uint64_t of = 0;  // whose failure `text` is of
    std::string text, other;
  };
  static Mine& mine() {
    thread_local Mine m;
    return m;
  }
  static uint64_t next() {  // (an address may be used again)
    static std::atomic<uint64_t> n{0};
    return ++n;
  }
  const uint64_t id_;
  mutable std::mutex lock_;
  std::string last_;
};

}  // namespace ecad
