// Joining a call's side streams when it returns before its own joins.
#pragma once

namespace cce {

// A call forks side streams off the caller's and joins them at its end.  Where it
// returns early (a launch failed), the kernels that run on them still read and write
// the call's buffers, which the caller frees in the order of its own stream: the
// guard makes that stream wait for them.  `Api` names the runtime's calls (true on
// success), so that the host test can stand in for them.
template <class Api>
class SideJoin {
 public:
  using Stream = typename Api::Stream;
  using Event = typename Api::Event;
  // `ev`: an event that nothing waits for between the fork and the join.
  SideJoin(Stream main, Event ev) : main_(main), ev_(ev) {}
  SideJoin(const SideJoin&) = delete;
  SideJoin& operator=(const SideJoin&) = delete;
  // From here on `side` has work of this call (it waits for the caller's stream already,
  // so it belongs to a capture that the caller's stream is in).
  void forked(Stream side) { side_[n_++] = side; }
  // The call has joined its streams itself.
  void joined() { n_ = 0; }
  ~SideJoin() {
    for (int i = 0; i < n_; ++i)
      if (!Api::record(ev_, side_[i]) || !Api::wait(main_, ev_)) Api::synchronize(side_[i]);
  }

 private:
  Stream main_;
  Event ev_;
  Stream side_[3];
  int n_ = 0;
};

}  // namespace cce
