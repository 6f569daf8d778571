"""Window attention and the paged cache without a GPU: descriptors, workspace sizes, and what the entry points refuse before they
launch anything."""

import ctypes
import re
import os

import pytest
import torch

from torch_mojo_backend_b200 import _lib, raw

FAKE = 0x7F0000000000  # never dereferenced: validation rejects the call first


def t4(ptr, shape, stride=None):
    if stride is None:
        b, h, s, d = shape
        stride = (h * s * d, s * d, d, 1)
    return _lib.pack_tensor4(ptr, *shape, *stride)


def window_fwd(**kw):
    q, k = kw.get("q_shape", (1, 4, 256, 64)), kw.get("k_shape", (1, 2, 256, 64))
    return _lib.window_fwd(t4(kw.get("q_ptr", FAKE), q, kw.get("q_stride")), t4(FAKE, k), t4(FAKE, kw.get("v_shape", k)), t4(FAKE, q, kw.get("out_stride")),
                           kw.get("lse", FAKE), kw.get("dtype", _lib.BF16), kw.get("causal", 1), kw.get("window", 64), kw.get("sinks", 4),
                           kw.get("scale", 0.125), 0, 0)


@pytest.mark.parametrize("how,expected", [
    (dict(window=0), _lib.ERR_UNSUPPORTED),
    (dict(window=-5), _lib.ERR_UNSUPPORTED),
    (dict(sinks=-1), _lib.ERR_UNSUPPORTED),
    (dict(causal=0), _lib.ERR_UNSUPPORTED),       # a window is causal
    (dict(causal=3), _lib.ERR_UNSUPPORTED),
    (dict(dtype=9), _lib.ERR_BAD_DTYPE),
    (dict(scale=0.0), _lib.ERR_UNSUPPORTED),
    (dict(q_shape=(1, 4, 256, 96)), _lib.ERR_UNSUPPORTED),
    (dict(q_shape=(1, 3, 256, 64)), _lib.ERR_BAD_SHAPE),
    (dict(v_shape=(1, 2, 255, 64)), _lib.ERR_BAD_SHAPE),
    (dict(q_shape=(1, 4, 0, 64)), _lib.ERR_BAD_SHAPE),
    (dict(q_stride=(65536, 16384, 64, 2)), _lib.ERR_BAD_STRIDE),
    (dict(out_stride=(65536, 64, 64, 1)), _lib.ERR_BAD_STRIDE),
    (dict(q_ptr=FAKE + 8), _lib.ERR_MISALIGNED),
    (dict(q_ptr=0), _lib.ERR_NULL),
    (dict(lse=0), _lib.ERR_NULL),
])
def test_window_forward_validates_before_launch(how, expected):
    before = _lib.launch_count()
    assert window_fwd(**how) == expected
    assert _lib.launch_count() == before


def test_window_backward_wants_its_own_workspace():
    """With few heads the sums of the blocks that share a tile with sinks come on top of the row statistics."""
    statistics = _lib.bwd_workspace_bytes(1, 4, 2, 8192, 128, _lib.BF16)
    size = lambda window, sinks, dtype=_lib.BF16, B=1: _lib.window_bwd_workspace_bytes(B, 4, 2, 8192, 8192, 128, dtype, window, sinks)
    assert size(512, 0) == statistics
    assert size(512, 4) > statistics and (size(512, 4) - statistics) % (2 * 128 * 128 * 4) == 0
    assert size(512, 4, _lib.F32) > statistics
    assert size(512, 200) > size(512, 4)                     # two tiles
    assert size(8192, 4) - statistics < size(512, 4)         # a window of everything has longer blocks to share with
    assert size(512, 4, B=512) == _lib.bwd_workspace_bytes(512, 4, 2, 8192, 128, _lib.BF16)   # enough blocks without
    assert size(0, 4) == 0 == size(512, -1) == _lib.window_bwd_workspace_bytes(1, 4, 0, 64, 64, 64, _lib.BF16, 8, 0)
    t = t4(FAKE, (1, 4, 8192, 128))
    k = t4(FAKE, (1, 2, 8192, 128))
    need, before = size(512, 4), _lib.launch_count()
    for ptr, n in ((0, need), (FAKE, need - 1), (FAKE, statistics), (FAKE + 16, need)):
        assert _lib.window_bwd(t, k, k, t, t, FAKE, t, k, k, ptr, n, _lib.BF16, 1, 512, 4, 0.1, 0, 0) == _lib.ERR_WORKSPACE
    assert _lib.window_bwd(t, k, k, t, t, FAKE, t, k, k, FAKE, need, _lib.BF16, 1, 0, 4, 0.1, 0, 0) == _lib.ERR_UNSUPPORTED
    assert _lib.launch_count() == before


def paged(**kw):
    fields = dict(k=FAKE, v=FAKE, k_scales=0, v_scales=0, table=FAKE, lengths=FAKE, new_lengths=0, pages=100, heads=2, page_size=16,
                  head_dim=64, batch=3, table_width=10, table_stride=10, dtype=_lib.BF16, bits=16)
    assert set(kw) <= set(fields)
    return _lib.pack_paged_kv(*{**fields, **kw}.values())


BAD_CACHES = [
    (dict(k=0), _lib.ERR_NULL), (dict(table=0), _lib.ERR_NULL), (dict(lengths=0), _lib.ERR_NULL),
    (dict(bits=4), _lib.ERR_NULL),                                     # no scales
    (dict(bits=8), _lib.ERR_UNSUPPORTED), (dict(dtype=_lib.F32), _lib.ERR_BAD_DTYPE), (dict(head_dim=96), _lib.ERR_UNSUPPORTED),
    (dict(page_size=8), _lib.ERR_UNSUPPORTED), (dict(page_size=48), _lib.ERR_UNSUPPORTED), (dict(page_size=8192), _lib.ERR_UNSUPPORTED),
    (dict(pages=0), _lib.ERR_BAD_SHAPE), (dict(heads=0), _lib.ERR_BAD_SHAPE), (dict(batch=0), _lib.ERR_BAD_SHAPE),
    (dict(batch=70000), _lib.ERR_BAD_SHAPE), (dict(table_width=0), _lib.ERR_BAD_SHAPE),
    (dict(table_width=(1 << 20) + 1, table_stride=1 << 21), _lib.ERR_BAD_SHAPE),   # more than 2^24 tokens
    (dict(pages=1 << 27), _lib.ERR_BAD_SHAPE),                         # 2^32 rows
    (dict(table_stride=9), _lib.ERR_BAD_STRIDE),
    (dict(k=FAKE + 8), _lib.ERR_MISALIGNED), (dict(lengths=FAKE + 2), _lib.ERR_MISALIGNED),
    (dict(bits=4, k_scales=FAKE, v_scales=FAKE + 4), _lib.ERR_MISALIGNED),
]


@pytest.mark.parametrize("how,expected", BAD_CACHES)
def test_every_call_on_a_paged_cache_validates_it_before_launch(how, expected):
    c, before = paged(**how), _lib.launch_count()
    D, B = how.get("head_dim", 64), how.get("batch", 3)
    q, k = t4(FAKE, (B, 4, 1, D)), t4(FAKE, (B, 2, 1, D))
    assert _lib.paged_attention(c, q, q, FAKE, 0, 0, 0.1, 0, 0, 0) == expected
    assert _lib.paged_append(c, k, k, q, q, FAKE, FAKE, 64, 100, False, 0, 0) == expected
    assert _lib.paged_gather(c, k, k, 0, 0) == expected
    assert _lib.launch_count() == before


def test_calls_on_a_paged_cache_validate_the_rest_before_launch():
    c, before = paged(), _lib.launch_count()
    q, k = t4(FAKE, (3, 4, 2, 64)), t4(FAKE, (3, 2, 2, 64))
    attend = lambda q=q, out=None, lse=FAKE, window=0, sinks=0, scale=0.1, longest=0: _lib.paged_attention(
        c, q, out or q, lse, window, sinks, scale, longest, 0, 0)
    assert _lib.paged_attention(c, q, q, FAKE, 0, 0, 0.1, 0, 0, 0, 0, FAKE + 4, 1 << 20) == _lib.ERR_MISALIGNED   # the workspace
    assert attend(lse=0) == _lib.ERR_NULL and attend(lse=FAKE + 1) == _lib.ERR_MISALIGNED
    assert attend(window=-1) == attend(sinks=-1) == attend(longest=-1) == attend(scale=-1.0) == _lib.ERR_UNSUPPORTED
    assert attend(t4(FAKE, (3, 3, 2, 64))) == _lib.ERR_BAD_SHAPE          # heads of q
    assert attend(t4(FAKE, (2, 4, 2, 64))) == _lib.ERR_BAD_SHAPE          # batch
    assert attend(t4(FAKE, (3, 4, 2, 128))) == _lib.ERR_BAD_SHAPE         # head dimension
    assert attend(t4(FAKE, (3, 64, 1 << 24, 64))) == _lib.ERR_BAD_SHAPE   # grid
    assert attend(out=t4(FAKE, (3, 4, 2, 64), (512, 64, 64, 1))) == _lib.ERR_BAD_STRIDE   # output rows overlap
    append = lambda k=k, v=k, q=q, q_out=q, cos=FAKE, sin=FAKE, R=64, positions=10: _lib.paged_append(
        c, k, v, q, q_out, cos, sin, R, positions, False, 0, 0)
    assert append(q_out=None) == append(q=None) == append(cos=0) == append(sin=0) == _lib.ERR_NULL
    assert append(R=8) == append(R=80) == append(R=-16) == _lib.ERR_UNSUPPORTED
    assert append(R=0) == _lib.ERR_UNSUPPORTED                             # queries and nothing that turns them
    assert append(positions=0) == _lib.ERR_BAD_SHAPE and append(cos=FAKE + 4) == _lib.ERR_MISALIGNED
    assert append(v=t4(FAKE, (3, 2, 3, 64))) == _lib.ERR_BAD_SHAPE
    assert append(k=t4(FAKE, (3, 2, 2, 64), (256, 128, 60, 1))) == _lib.ERR_BAD_STRIDE
    assert append(q_out=t4(FAKE, (3, 4, 2, 64), (0, 128, 64, 1))) == _lib.ERR_BAD_STRIDE
    gather = lambda k, v: _lib.paged_gather(c, k, v, 0, 0)
    assert gather(k, t4(FAKE, (3, 2, 3, 64))) == _lib.ERR_BAD_SHAPE and gather(None, k) == _lib.ERR_NULL
    assert gather(t4(FAKE, (3, 2, 1 << 25, 64)), k) == _lib.ERR_BAD_SHAPE
    assert _lib.launch_count() == before


def test_the_workspace_of_attention_over_a_paged_cache():
    need = _lib.paged_attention_workspace_bytes
    assert need(1, 8, 1, 1, 128, 100000) == 16 * 8 * 132 * 4            # 16 clusters, 8 rows, their maxima and sums
    assert need(1, 8, 1, 4, 64, 100000) == 16 * 2 * 16 * 68 * 4         # two tiles of 16 rows
    assert need(1, 8, 1, 1, 128, 4096) == need(64, 32, 8, 1, 128, 100000) == 0
    assert need(1, 3, 2, 1, 128, 100000) == need(0, 8, 1, 1, 128, 100000) == need(1, 8, 0, 1, 128, 100000) == 0
    assert need(1, 8, 1, 1, 96, 100000) == need(1, 8, 1, 1 << 40, 64, 100000) == need(1 << 62, 8, 1, 1, 64, 1 << 62) == 0


def test_valid_calls_without_a_gpu_report_an_error():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present; this checks the no-GPU failure mode")
    q, k = t4(FAKE, (3, 4, 2, 64)), t4(FAKE, (3, 2, 2, 64))
    for rc in (window_fwd(), _lib.paged_attention(paged(), q, q, FAKE, 0, 0, 0.1, 0, 0, 0),
               _lib.paged_append(paged(), k, k, q, q, FAKE, FAKE, 64, 100, False, 0, 0), _lib.paged_gather(paged(), k, k, 0, 0)):
        assert rc in (_lib.ERR_CUDA, _lib.ERR_UNSUPPORTED)


def test_the_descriptor_is_the_headers():
    assert ctypes.sizeof(_lib.PagedCache) == len(paged()) == 7 * 8 + 7 * 8 + 2 * 4
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "b200fa.h")).read()
    body = re.search(r"typedef struct b200fa_paged_kv \{(.*?)\}", header, re.S).group(1)
    names = [n.strip(" *") for line in body.split(";") for n in re.sub(r"^\s*(const )?(void|int32_t|int64_t|int)\b", "", line.strip()).split(",") if n.strip()]
    assert names == [n for n, _ in _lib.PagedCache._fields_]


def test_status_of_a_bad_index():
    assert _lib.status_to_error(0x42490003) == _lib.ERR_BAD_INDEX and "out of range" in _lib.strerror(_lib.ERR_BAD_INDEX)


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 2, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA"):
        raw.window_fwd(q, q, q, window=2)
    with pytest.raises(RuntimeError, match="CUDA"):
        raw.window_bwd(q, q, q, q, q, torch.zeros(1, 2, 4), window=2)
    cache = raw.PagedKV.empty(4, 2, 16, 64, device="cpu")
    i = torch.zeros(1, 2, dtype=torch.int32)
    for call in (lambda: raw.paged_attention(q, cache, i, i[0]), lambda: raw.paged_append(q, q, cache, i, i[0]),
                 lambda: raw.paged_gather(cache, i, i[0, :1], 3)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_pools_of_codes():
    c = raw.PagedKV.empty(5, 3, 32, 128, dtype=torch.float16, bits=4, device="cpu")
    assert c.k.shape == (5, 3, 32, 64) and c.k.dtype == torch.uint8 and c.v_scales.shape == (5, 3, 32, 4, 2) and c.dtype == torch.float16
    with pytest.raises(NotImplementedError):
        raw.PagedKV.empty(5, 3, 32, 128, bits=8, device="cpu")


def test_window_attention_refuses_from_the_forward(host_backed_mojo):
    import torch_mojo_backend_b200 as tmb

    q = torch.zeros(1, 4, 8, 64, dtype=torch.bfloat16).to("mojo")
    k = torch.zeros(1, 2, 8, 64, dtype=torch.bfloat16).to("mojo")
    for how in (dict(window=0), dict(window=2.0), dict(window=True), dict(window=3, sinks=-1), dict(window=3, scale=-1.0)):
        with pytest.raises(NotImplementedError):
            tmb.window_attention(q, q, q, **how)
    with pytest.raises(NotImplementedError):
        tmb.window_attention(q, k, k, 3)                      # needs enable_gqa
    with pytest.raises(NotImplementedError):
        tmb.window_attention(q, q, torch.zeros(1, 4, 8, 64, dtype=torch.bfloat16), 3)   # a CPU tensor
    assert host_backed_mojo.calls == []


def test_a_paged_cache_refuses_what_the_kernels_do_not_serve(mojo_registered):
    for how in (dict(head_dim=96), dict(page_size=24), dict(dtype=torch.float32), dict(bits=8)):
        args = dict(pages=2, kv_heads=1, page_size=16, head_dim=64)
        with pytest.raises((NotImplementedError, RuntimeError)) as err:
            mojo_registered.PagedKVCache(**{**args, **how})
        assert err.type is NotImplementedError


def test_the_shares_of_a_paged_call_are_refused_before_a_device_is_asked():
    good = dict(B=2, Hq=8, Hkv=2, S=1, D=128, dtype=_lib.BF16, bits=16, longest=1000)
    for how, code in ((dict(B=0), _lib.ERR_BAD_SHAPE), (dict(Hq=7), _lib.ERR_BAD_SHAPE), (dict(Hkv=0), _lib.ERR_BAD_SHAPE), (dict(S=0), _lib.ERR_BAD_SHAPE),
                      (dict(longest=0), _lib.ERR_BAD_SHAPE), (dict(longest=1 << 25), _lib.ERR_BAD_SHAPE), (dict(S=1 << 40), _lib.ERR_BAD_SHAPE),
                      (dict(D=96), _lib.ERR_UNSUPPORTED), (dict(bits=8), _lib.ERR_UNSUPPORTED), (dict(dtype=_lib.F32), _lib.ERR_BAD_DTYPE)):
        with pytest.raises(_lib.B200FAError) as err:
            _lib.paged_attention_shares(**{**good, **how})
        assert err.value.code == code


def test_calls_of_few_keys_do_not_ask_for_a_workspace(monkeypatch):
    """The query costs a short call a tenth of its time on the host: tables of fewer keys than any workspace is for go without it."""
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "b200fa.h")).read()
    for name, value in (("PAGED_TEAM_KEYS", _lib.PAGED_TEAM_KEYS), ("APPEND_CLEAR", _lib.APPEND_CLEAR)):
        assert int(re.search(rf"#define B200FA_{name} (\w+)", header).group(1), 0) == value
    need = _lib.paged_attention_workspace_bytes
    assert need(1, 8, 1, 1, 128, _lib.PAGED_TEAM_KEYS - 1) == 0 < need(1, 8, 1, 1, 128, _lib.PAGED_TEAM_KEYS)
    asked = []
    monkeypatch.setattr(_lib, "paged_attention_workspace_bytes", lambda *a: asked.append(a) or 0)
    monkeypatch.setattr(_lib, "paged_attention", lambda *a: _lib.OK)
    monkeypatch.setattr(raw, "_stream_and_device", lambda t: (0, 0))
    q = torch.zeros(2, 4, 3, 64, dtype=torch.bfloat16)

    def call(width, **how):
        monkeypatch.setattr(raw, "_paged", lambda *a: (b"", q.dtype, 2, 64, q.device, 16 * width))
        raw.paged_attention(q, None, None, None, **how)
        got = asked[:]
        asked.clear()
        return got

    assert call(511) == [] == call(511, longest=100) == call(511, window=20)
    assert call(512) == [(2, 4, 2, 3, 64, 8192)] and call(600, longest=9000) == [(2, 4, 2, 3, 64, 9000)]
    assert call(600, longest=10000) == [(2, 4, 2, 3, 64, 9600)] and call(600, window=8200, sinks=4) == [(2, 4, 2, 3, 64, 8207)]


@pytest.mark.parametrize("which", ["query", "key", "value", "rotary"])
def test_a_paged_cache_refuses_tensors_that_want_gradients(host_backed_mojo, which, monkeypatch):
    """Their gradients would be lost without a word: nothing goes back through the pages."""
    import torch_mojo_backend_b200 as tmb

    cache = tmb.PagedKVCache.__new__(tmb.PagedKVCache)   # (its pages are CUDA memory)
    cache.kv = cache._status = None
    reached = []
    monkeypatch.setattr(raw, "paged_append", lambda *a, **how: reached.append("append"))
    monkeypatch.setattr(raw, "paged_attention", lambda *a, **how: reached.append("attention") or (torch.zeros(1), torch.zeros(1)))
    monkeypatch.setattr(tmb.PagedKVCache.attention.__globals__["TorchMojoTensor"], "_from_cuda", staticmethod(lambda t: t))
    make = lambda *shape, want=False: torch.zeros(*shape).to("mojo").requires_grad_(want)   # noqa: E731
    i = torch.zeros(1, 1, dtype=torch.int32).to("mojo")
    q, k, v = (make(1, 2, 1, 64, want=which == n) for n in ("query", "key", "value"))
    angles = make(16, 32, want=which == "rotary"), make(16, 32)

    def calls():
        cache.append(k, v, i, i, rotary=angles, query=q)
        if which == "query":
            cache.attention(q, i, i)

    with pytest.raises(NotImplementedError, match=f"{which} requires a gradient"):
        cache.append(k, v, i, i, rotary=angles, query=q)
    if which == "query":
        with pytest.raises(NotImplementedError, match="query requires a gradient"):
            cache.attention(q, i, i)
    assert reached == []
    with torch.no_grad():
        calls()
    with torch.inference_mode():
        calls()
    assert reached == (["append", "attention"] if which == "query" else ["append"]) * 2


def test_a_bad_index_waits_for_the_check_that_asks_for_it(host_backed_mojo):
    from torch_mojo_backend_b200 import flash_ops

    word = flash_ops._status_words[0]._cuda_view()
    word.fill_(0x42490006)
    flash_ops.check_status(0, bad_index=False)       # (what the host pipeline asks)
    with pytest.raises(_lib.B200FAError) as err:
        flash_ops.check_status(0)
    assert err.value.code == _lib.ERR_BAD_INDEX
    flash_ops.check_status(0)
    word.fill_(0x57410320)
    with pytest.raises(_lib.B200FAError) as err:
        flash_ops.check_status(0, bad_index=False)
    assert err.value.code == _lib.ERR_TIMEOUT
    flash_ops.check_status(0)
