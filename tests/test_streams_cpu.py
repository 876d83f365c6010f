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


class _Noted(torch.autograd.Function):
    """A Unit's part in this: the forward notes the block it runs in, the backward joins."""

    @staticmethod
    def forward(ctx, x):
        from keypoints_amd import runtime
        ctx.forked = runtime.forked_from()
        return x * 2

    @staticmethod
    def backward(ctx, g):
        from keypoints_amd import runtime
        runtime.join_after_backward(ctx.forked)
        return g * 2


def test_a_checkpointed_forward_in_a_side_block_is_joined(monkeypatch):
    """torch.utils.checkpoint runs the forward again inside the backward, on the side stream but in no block: its backward's work on that stream
    is still joined to the stream the block was forked from (the optimizer reads it there).  A stream of one's own is not."""
    from torch.utils.checkpoint import checkpoint
    from keypoints_amd import runtime
    pool = _Pool()
    monkeypatch.setattr(torch.cuda, 'Stream', pool.Stream)
    monkeypatch.setattr(torch.cuda, 'stream', pool.stream)
    monkeypatch.setattr(torch.cuda, 'current_stream', lambda *a: pool.now)
    for name in ('_side_streams', '_held', '_forks'):
        monkeypatch.setattr(runtime, name, {})
    monkeypatch.setattr(runtime, '_used', set())
    capturing = set()   # streams that a capture is in progress on
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: pool.now.stream_id in capturing)

    class OnDevice:
        is_cuda = True

    main = pool.now
    for reentrant in (True, False):
        x = torch.ones(3, requires_grad=True)
        with runtime.fork('chain', OnDevice()) as side:
            with side:
                chain = pool.now
                y = checkpoint(_Noted.apply, x, use_reentrant=reentrant)
        for caught in (set(), {main.stream_id, chain.stream_id}):
            capturing.clear()
            capturing.update(caught)
            pool.now = chain                      # (the engine runs a node's backward on the stream of its forward)
            pool.waits.clear()
            y.sum().backward(retain_graph=True)
            pool.now = main
            assert (main.stream_id, chain.stream_id) in pool.waits, (reentrant, caught)
    # a capture of one's own on a stream that the pool hands out again: the old parent is not drawn into it
    capturing.clear()
    capturing.add(chain.stream_id)
    x = torch.ones(3, requires_grad=True)
    with pool.stream(chain):
        y = checkpoint(_Noted.apply, x, use_reentrant=True)
        pool.waits.clear()
        y.sum().backward()
    assert pool.waits == []
