"""Window attention and the paged cache through the `mojo` device (``-m gpu``): the same kernels as the calls in ``raw``, so the same
bits, with autograd, streams and the device's status word around them."""

import pytest
import torch

import torch_mojo_backend_b200 as tmb
from tests.test_gpu_window import TL, BR, inputs, run_both
from torch_mojo_backend_b200 import _lib, raw

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def mojo():
    tmb.register_mojo_devices()


def leaves(*ts):
    return [tmb.from_cuda(t).requires_grad_() for t in ts]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("Sq,Sk,causal", [(500, 500, TL), (200, 700, BR)])
def test_window_attention_and_its_gradients_are_the_kernels(Sq, Sk, causal, dtype):
    q, k, v, grad = inputs(1, 2, 4, 2, Sq, Sk, 64, dtype)
    want = run_both(q, k, v, grad, causal, 100, 3)
    mq, mk, mv = leaves(q, k, v)
    out, lse = tmb.window_attention(mq, mk, mv, 100, sinks=3, bottom_right=causal == BR, enable_gqa=True, return_lse=True)
    assert out.requires_grad and not lse.requires_grad
    out.backward(tmb.from_cuda(grad))
    torch.mojo.synchronize()
    for name, got in (("out", out.detach()), ("lse", lse), ("dq", mq.grad), ("dk", mk.grad), ("dv", mv.grad)):
        assert torch.equal(tmb.to_cuda(got), want[name]), name


def test_window_attention_of_a_fused_projection_keeps_its_layout():
    B, H, S, D = 2, 4, 300, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    fused = torch.randn(B, S, 3 * H * D, generator=g, device="cuda").bfloat16()
    views = [t.unflatten(2, (H, D)).transpose(1, 2) for t in fused.split(H * D, 2)]
    grad = torch.randn(B, S, H, D, generator=g, device="cuda").bfloat16().transpose(1, 2)
    want = run_both(*(t.contiguous() for t in views), grad.contiguous(), TL, 64, 2)
    q, k, v = leaves(*views)
    out = tmb.window_attention(q, k, v, 64, sinks=2)
    assert tmb.to_cuda(out.detach()).transpose(1, 2).is_contiguous()
    grads = torch.autograd.grad(out, (q, k, v), tmb.from_cuda(grad))
    assert torch.equal(tmb.to_cuda(out.detach()), want["out"])
    for name, got in zip(("dq", "dk", "dv"), grads):
        assert torch.equal(tmb.to_cuda(got), want[name]) and tmb.to_cuda(got).transpose(1, 2).is_contiguous()


def test_the_same_tensor_as_key_and_value_and_a_result_that_nobody_differentiates():
    q, k, _, grad = inputs(4, 1, 2, 2, 200, 200, 64, torch.bfloat16)
    want = run_both(q, k, k, grad, TL, 50, 0)
    mq, mk = leaves(q, k)
    out = tmb.window_attention(mq, mk, mk, 50)
    out.backward(tmb.from_cuda(grad))
    torch.mojo.synchronize()
    assert torch.equal(tmb.to_cuda(mk.grad), want["dk"] + want["dv"])
    with torch.no_grad():
        assert torch.equal(tmb.to_cuda(tmb.window_attention(mq, mk, mk, 50)), want["out"])


def test_autocast_casts_the_tensors():
    q, k, v, _ = inputs(6, 1, 2, 2, 200, 200, 64, torch.float32)
    want, _ = raw.window_fwd(q.bfloat16(), k.bfloat16(), v.bfloat16(), window=50)
    mq, mk, mv = leaves(q, k, v)
    with torch.autocast("mojo", dtype=torch.bfloat16):
        out = tmb.window_attention(mq, mk, mv, 50)
    assert out.dtype == torch.bfloat16 and torch.equal(tmb.to_cuda(out.detach()), want)
    out.backward(torch.ones(out.shape, dtype=torch.bfloat16).to("mojo"))
    assert mq.grad.dtype == torch.float32


def test_a_training_step_on_a_side_stream_and_in_a_graph():
    """The backward runs on the stream of the forward, whichever thread the engine calls it from."""
    q, k, v, grad = inputs(5, 1, 4, 2, 1500, 1500, 128, torch.bfloat16)
    want = run_both(q, k, v, grad, TL, 200, 4)
    mq, mk, mv = leaves(q, k, v)
    g = tmb.from_cuda(grad)

    def step():
        out = tmb.window_attention(mq, mk, mv, 200, sinks=4, enable_gqa=True)
        return [tmb.to_cuda(t) for t in (out.detach(), *torch.autograd.grad(out, (mq, mk, mv), g))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    for name, t in zip(("out", "dq", "dk", "dv"), got):
        assert torch.equal(t, want[name]), name
    alive = tmb.window_attention(mq, mk, mv, 200, sinks=4, enable_gqa=True)   # an eager graph of the same leaves
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for t in got:
        t.zero_()
    q.mul_(0.5)
    graph.replay()
    want = run_both(q, k, v, grad, TL, 200, 4)
    for name, t in zip(("out", "dq", "dk", "dv"), got):
        assert torch.equal(t, want[name]), name
    assert alive.requires_grad


@pytest.mark.parametrize("how", ["one tensor twice", "views of one", "twice into a grad", "with another operator"])
def test_what_the_engine_adds_on_a_side_stream_and_in_a_graph(how):
    """Sums of gradients and gradients of views are the engine's, on its own thread."""
    q, k, v, grad = inputs(7, 1, 4, 4, 2048, 2048, 128, torch.bfloat16)
    g = tmb.from_cuda(grad)
    if how == "views of one":
        fused = leaves(torch.stack([q, k, v]))
        call = lambda: tmb.window_attention(*(fused[0][i] for i in range(3)), 200)   # noqa: E731
    else:
        fused = leaves(q, k, v)
        mk, mv = fused[1], fused[1 if how == "one tensor twice" else 2]
        call = lambda: tmb.window_attention(fused[0], mk, mv, 200)   # noqa: E731
    if how == "with another operator":
        first = call
        call = lambda: torch.nn.functional.scaled_dot_product_attention(first(), mk, mv, is_causal=True)   # noqa: E731

    def step():
        for t in fused:
            t.grad = None
        with torch.autograd.set_multithreading_enabled(how != "with another operator"):
            for _ in range(2 if how == "twice into a grad" else 1):
                call().backward(g)
        return [tmb.to_cuda(t.grad).clone() for t in fused if t.grad is not None]

    want = step()
    torch.cuda.synchronize()
    busy = torch.ones(8192, 8192, device="cuda")
    side = torch.cuda.Stream()
    for on in (side, torch.cuda.default_stream()):   # the stream that is behind
        torch.cuda.synchronize()
        with torch.cuda.stream(on):
            for _ in range(4):
                busy @ busy
        with torch.cuda.stream(side):
            got = step()
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for t in got:
        t.zero_()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    streams = []   # the engine's thread is back on its own
    fused[0].register_hook(lambda _: streams.append(torch.cuda.current_stream()))
    got = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and set(streams) == {torch.cuda.default_stream()}


@pytest.mark.parametrize("bits", [16, 4])
def test_paged_cache_on_the_device(bits):
    B, Hq, Hkv, D, page = 2, 8, 2, 128, 16
    cache = tmb.PagedKVCache(12, Hkv, page, D, dtype=torch.float16, bits=bits)
    assert cache.dtype == torch.float16
    table = torch.tensor([[3, 5, 7, 9, 11, 0], [1, 2, 4, 6, 8, 10]], dtype=torch.int32)
    lengths = torch.tensor([70, 33], dtype=torch.int32)
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn(B, h, 70, D, generator=g, device="cuda").half() for h in (Hq, Hkv, Hkv))
    angle = torch.rand(96, 64, device="cuda", generator=g)
    rotary = angle.cos(), angle.sin()
    plain = raw.PagedKV.empty(12, Hkv, page, D, dtype=torch.float16, bits=bits)
    tq = raw.paged_append(k, v, plain, table.cuda(), lengths.cuda(), new_lengths=lengths.cuda(), rotary=rotary, q=q)
    want, want_lse = raw.paged_attention(tq, plain, table.cuda(), lengths.cuda(), new_lengths=lengths.cuda(), window=20, sinks=1)
    gk, gv = raw.paged_gather(plain, table.cuda(), lengths.cuda(), 80)
    m = [t.to("mojo") for t in (table, lengths)]
    turned = cache.append(tmb.from_cuda(k), tmb.from_cuda(v), *m, new_lengths=m[1], rotary=[tmb.from_cuda(t) for t in rotary],
                          query=tmb.from_cuda(q))
    out, lse = cache.attention(turned, *m, new_lengths=m[1], window=20, sinks=1, return_lse=True)
    mk, mv = cache.gather(*m, 80)
    torch.mojo.synchronize()
    for got, ref in ((turned, tq), (out, want), (lse, want_lse), (mk, gk), (mv, gv)):
        assert torch.equal(tmb.to_cuda(got), ref)
    with pytest.raises(RuntimeError, match="mojo tensor"):
        cache.attention(tq, *m)
    # an index out of range surfaces where the device is synchronised
    cache.attention(turned, m[0], torch.tensor([97, 33], dtype=torch.int32).to("mojo"))
    with pytest.raises(_lib.B200FAError) as err:
        torch.mojo.synchronize()
    assert err.value.code == _lib.ERR_BAD_INDEX
    again = cache.attention(turned, *m, new_lengths=m[1], window=20, sinks=1)
    torch.mojo.synchronize()
    assert torch.equal(tmb.to_cuda(again), want)


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 64)])
def test_a_bad_index_stops_no_other_call(dtype, D):
    """The device's status word also stops kernels whose waits have run out: an index out of range of a paged call is not that."""
    q, k, v, grad = inputs(8, 1, 4, 2, 700, 700, D, dtype)
    cache = tmb.PagedKVCache(4, 2, 16, 64)
    cache.kv.k.zero_(), cache.kv.v.zero_()
    table = torch.arange(4, dtype=torch.int32).view(1, 4).to("mojo")
    lengths = [torch.tensor([n], dtype=torch.int32).to("mojo") for n in (65, 64)]   # one more than there is room for; all of them
    query = torch.zeros(1, 2, 1, 64, dtype=torch.bfloat16).to("mojo")

    def calls():
        got = []
        for call in (lambda *t: tmb.window_attention(*t, 100, sinks=3, enable_gqa=True),
                     lambda *t: torch.nn.functional.scaled_dot_product_attention(*t, is_causal=True, enable_gqa=True)):
            t = leaves(q, k, v)
            out = call(*t)
            out.backward(tmb.from_cuda(grad))
            got += [tmb.to_cuda(x).clone() for x in (out.detach(), *(x.grad for x in t))]
        return got

    want = calls()
    torch.mojo.synchronize()
    assert torch.isnan(tmb.to_cuda(cache.attention(query, table, lengths[0]))).all()
    got = calls()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert not tmb.to_cuda(cache.attention(query, table, lengths[1])).any()
    with pytest.raises(_lib.B200FAError) as err:
        torch.mojo.synchronize()
    assert err.value.code == _lib.ERR_BAD_INDEX
    torch.mojo.synchronize()


def test_a_wait_that_runs_out_takes_a_bad_indexs_place():
    status = torch.tensor([0x42490006], dtype=torch.int32, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    assert _lib.selftest_wait_timeout(status.data_ptr(), 1_000_000, stream, 0) == _lib.OK
    torch.cuda.synchronize()
    assert _lib.status_to_error(int(status) & 0xFFFFFFFF) == _lib.ERR_TIMEOUT
    # and an index out of range does not take its
    pool = raw.PagedKV.empty(1, 1, 16, 64)
    held = int(status)
    raw.paged_gather(pool, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.full((1,), 17, dtype=torch.int32, device="cuda"), 3,
                     status=status)
    torch.cuda.synchronize()
    assert int(status) == held


class Held(torch.autograd.Function):
    """A CPU tensor that stands for `held` on the device: its own gradient is the caller's thread's business."""

    @staticmethod
    def forward(ctx, x, held):
        return held.detach()

    @staticmethod
    def backward(ctx, grad):
        return torch.zeros(1), None


@pytest.mark.parametrize("fails", [True, False])
def test_a_captured_backward_that_fails_or_ends_on_another_thread(fails):
    """It leaves the engine's thread on the stream that it found there: backwards behind it are ordered with the default stream."""
    q, k, v, grad = inputs(9, 1, 4, 4, 1024, 1024, 64, torch.bfloat16)
    g = tmb.from_cuda(grad)

    def step(call):
        t = leaves(q, k, v)
        streams = []
        t[0].register_hook(lambda _: streams.append(torch.cuda.current_stream()))
        call(*t).backward(g)
        return [tmb.to_cuda(x.grad).clone() for x in t], streams

    calls = (lambda *t: tmb.window_attention(*t, 100), lambda *t: torch.nn.functional.scaled_dot_product_attention(*t, is_causal=True))
    want = [step(call)[0] for call in calls]
    held = [tmb.from_cuda(t) for t in (q, k, v)]
    x, called = torch.zeros(1, requires_grad=True), []

    def hook(_):
        called.append(1)
        if fails:
            raise ValueError("on purpose")

    x.register_hook(hook)
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph):
            tmb.window_attention(Held.apply(x, held[0]), *held[1:], 100).backward(g)
    except ValueError:
        assert fails
    assert called
    torch.cuda.synchronize()
    for call, ref in zip(calls[::-1], want[::-1]):
        got, streams = step(call)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, ref)) and streams == [torch.cuda.default_stream()]


@pytest.mark.parametrize("bits", [16, 4])
def test_paged_cache_on_a_side_stream(bits):
    """append, attention and gather are ordered on the current stream, whatever the default one is doing."""
    g = torch.Generator(device="cuda").manual_seed(1)
    lengths = torch.tensor([9000, 700], dtype=torch.int32)
    table = torch.arange(2 * 141, dtype=torch.int32).view(2, 141)
    q, k, v = (torch.randn(2, h, 9000, 64, generator=g, device="cuda").bfloat16() for h in (2, 1, 1))
    row = torch.randn(2, 2, 1, 64, generator=g, device="cuda").bfloat16()
    busy = torch.ones(8192, 8192, device="cuda")

    def run():
        cache = tmb.PagedKVCache(2 * 141, 1, 64, 64, bits=bits)
        m = [t.to("mojo") for t in (table, lengths)]
        cache.append(tmb.from_cuda(k), tmb.from_cuda(v), *m, new_lengths=m[1])
        out, lse = cache.attention(tmb.from_cuda(row), *m, return_lse=True)   # (its workspace is the stream's too)
        return [tmb.to_cuda(t) for t in (out, lse, *cache.gather(*m, 9000))]

    want = run()
    torch.mojo.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for on in (side, torch.cuda.default_stream()):   # the stream that is behind
        with torch.cuda.stream(on):
            for _ in range(4):
                busy @ busy
        with torch.cuda.stream(side):
            got = run()
        side.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.mojo.synchronize()


def test_a_bad_index_does_not_end_a_host_pass():
    """The pipeline answers for its own kernels; an index out of range of a paged call is told by the device's synchronize."""
    g = torch.Generator().manual_seed(2)
    q, k, v = (tmb.pinned_empty((2, 2, 300, 64), torch.bfloat16) for _ in range(3))
    for t in (q, k, v):
        t.copy_(torch.randn(t.shape, generator=g).bfloat16())
    pipe = tmb.HostAttentionPipeline(0, piece_bytes=1 << 20)
    want = pipe.run(q, k, v, is_causal=True)[0]
    pipe.synchronize()
    want = want.clone()
    cache = tmb.PagedKVCache(2, 1, 16, 64)
    i = torch.full((1, 1), 9, dtype=torch.int32).to("mojo")
    cache.attention(torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16).to("mojo"), i, torch.ones(1, dtype=torch.int32).to("mojo"))
    got = pipe.run(q, k, v, is_causal=True)[0]
    pipe.synchronize()
    assert torch.equal(got, want)
    with pytest.raises(_lib.B200FAError) as err:
        torch.mojo.synchronize()
    assert err.value.code == _lib.ERR_BAD_INDEX


@pytest.mark.parametrize("how", ["window", "paged", "dense"])
def test_a_first_call_in_a_capture(how, monkeypatch):
    """The device's status word is there before: the graph neither makes it nor wipes what was reported."""
    from torch_mojo_backend_b200 import flash_ops, tensor

    q, k, v, _ = inputs(10, 1, 2, 2, 256, 256, 64, torch.bfloat16)
    words = {}
    monkeypatch.setattr(flash_ops, "_status_words", words)
    monkeypatch.setattr(tensor, "_used", set(), raising=False)
    t = [tmb.from_cuda(x) for x in (q, k, v)]
    cache = tmb.PagedKVCache(4, 2, 16, 64)
    cache.kv.k.zero_(), cache.kv.v.zero_()
    table, lengths = (tmb.from_cuda(torch.tensor(x, dtype=torch.int32, device="cuda")) for x in ([[0, 1, 2, 3]], [50]))
    row = tmb.from_cuda(q[:, :, :1].contiguous())
    call = {"window": lambda: tmb.window_attention(*t, 30), "paged": lambda: cache.attention(row, table, lengths),
            "dense": lambda: torch.nn.functional.scaled_dot_product_attention(*t, is_causal=True)}[how]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    word = words[0]._cuda_view()
    word.fill_(0x42490001)
    graph.replay()
    assert int(word) == 0x42490001
    word.zero_()
    assert torch.equal(tmb.to_cuda(out), tmb.to_cuda(call()))
    torch.mojo.synchronize()
