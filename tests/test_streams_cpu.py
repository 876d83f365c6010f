"""CPU: which stream the runtime's side blocks are joined to, on streams as torch hands them out."""
import torch


class _Pool:
    """Streams as torch hands them out: a pool of 32 in turn, equal where they are the same stream of the device."""

    def __init__(self):
        self.made, self.waits, self.now = 0, [], None
        pool = self

        class Stream:
            def __init__(self, device=None, stream_id=None):
                if stream_id is None:
                    pool.made += 1
                    stream_id = 1 + (pool.made - 1) % 32
                self.stream_id, self.device = stream_id, torch.device('cuda', 0)

            def __eq__(self, other):
                return self.stream_id == other.stream_id

            def __hash__(self):
                return self.stream_id

            def wait_stream(self, other):
                pool.waits.append((self.stream_id, other.stream_id))

        class On:
            def __init__(self, stream):
                self.stream = stream

            def __enter__(self):
                self.back, pool.now = pool.now, self.stream

            def __exit__(self, *exc):
                pool.now = self.back

        self.Stream, self.stream, self.now = Stream, On, Stream(stream_id=0)


def test_a_stream_from_the_pool_that_was_once_a_side_stream(monkeypatch):
    """An application's (or a capture's) stream may be one that was taken as a side stream before: a backward on it must not make that side
    stream's parent wait -- inside a capture this drew a stream of its own into it that nothing joined."""
    from keypoints_amd import runtime
    pool = _Pool()
    monkeypatch.setattr(torch.cuda, 'Stream', pool.Stream)
    monkeypatch.setattr(torch.cuda, 'stream', pool.stream)
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda *a: pool.now)
    monkeypatch.setattr(runtime, '_side_streams', {})
    monkeypatch.setattr(runtime, '_used', set())
    monkeypatch.setattr(runtime, '_held', {})

    class OnDevice:
        is_cuda = True

    main = pool.now
    with runtime.fork('chain', OnDevice()) as side:
        with side:
            chain, inside = pool.now, runtime.forked_from()
    assert inside == main and runtime.forked_from() is None and chain != main
    pool.now = chain                                  # a Unit's backward behind that forward: its parent waits for it
    pool.waits.clear()
    runtime.join_after_backward(inside)
    assert pool.waits == [(main.stream_id, chain.stream_id)]
    pool.now = main

    mine = pool.Stream()
    while mine != chain:                              # the pool comes round
        mine = pool.Stream()
    with pool.stream(mine):                           # a forward and backward on a stream of one's own
        forked = runtime.forked_from()
        pool.waits.clear()
        runtime.join_after_backward(forked)
        assert pool.waits == [] and not runtime.nested_fork_under_capture(forked)
        pool.made = mine.stream_id - 1                # the next one of the pool is the current stream
        assert runtime.side_stream('wgrad') != mine
