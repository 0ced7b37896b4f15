"""qwn_prompt_attention on the GPU: packed prompts against the formula in 64 bits."""
from __future__ import annotations

import ctypes as C

import pytest

pytestmark = pytest.mark.gpu

KINDS = ["bf16", "f16", "f32"]


def _rows(torch, kind, lens, hq, hk, seed=0, pad=0):
    from promptmath import HEAD, TYPES
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn((sum(lens) + pad, hq + 2 * hk, HEAD), device="cuda", generator=g)
    x[:, :hq + hk, ::37] *= 6  # some channels are larger, so that some rows see little beside one token
    return x.to(TYPES[kind])


def _begin(torch, lens, offset=0):
    b = [offset]
    for n in lens:
        b.append(b[-1] + n)
    return torch.tensor(b, dtype=torch.int32, device="cuda")


def _run(torch, x, lens, hq, hk, kind, causal=True, window=0, out=None, begin="yes", **more):
    import qwanto_b200 as qb
    from promptmath import HEAD, TYPE_ID
    rows, wide = x.shape[0], x.shape[1] * HEAD
    if out is None:
        out = torch.full((rows, hq, HEAD), 7.0, dtype=x.dtype, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    flat = x.view(rows, -1)
    qb.prompt_attention(flat, flat[:, hq * HEAD:], flat[:, (hq + hk) * HEAD:], out, rows, TYPE_ID[kind], hq, hk,
                        num_seqs=len(lens), row_begin=_begin(torch, lens) if begin == "yes" else begin, causal=causal,
                        window=window, query_stride=wide, key_stride=wide, value_stride=wide, status=status, **more)
    torch.cuda.synchronize()
    assert int(status) == 0
    return out


def _check(torch, out, x, lens, hq, hk, kind, causal=True, window=0, scale=0.0, at=0):
    from promptmath import assert_near, attend, seen
    for i, n in enumerate(lens):
        y = x[at:at + n]
        want, tol = attend(y[:, :hq], y[:, hq:hq + hk], y[:, hq + hk:], seen(0, n, n, causal, window), scale, kind)
        assert_near(out[at:at + n], want, tol, f"sequence {i} of {lens}")
        at += n


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens", [[1], [2, 127, 1], [128], [129, 64], [300, 1, 65], [515]])
@pytest.mark.parametrize("heads", [(1, 1), (12, 2), (8, 1)])
def test_prompts(cuda, kind, lens, heads):
    torch, (hq, hk) = cuda, heads
    x = _rows(torch, kind, lens, hq, hk, seed=len(lens) + hq)
    _check(torch, _run(torch, x, lens, hq, hk, kind), x, lens, hq, hk, kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("window", [1, 2, 100, 128, 257, 4000])
def test_windows(cuda, kind, window):
    torch, lens = cuda, [1, 333, 700]
    x = _rows(torch, kind, lens, 4, 2, seed=window)
    _check(torch, _run(torch, x, lens, 4, 2, kind, window=window), x, lens, 4, 2, kind, window=window)


@pytest.mark.parametrize("kind", KINDS)
def test_not_causal(cuda, kind):
    torch, lens = cuda, [1, 130, 400, 128]
    x = _rows(torch, kind, lens, 6, 2, seed=5)
    _check(torch, _run(torch, x, lens, 6, 2, kind, causal=False), x, lens, 6, 2, kind, causal=False)


@pytest.mark.parametrize("kind", KINDS)
def test_enough_rows_for_two_tiles_per_block(cuda, kind):
    """More than an SM's worth of row tiles each: 256 rows per block of threads for 16-bit rows."""
    torch, lens = cuda, [1500, 77, 3, 900, 256]
    x = _rows(torch, kind, lens, 32, 8, seed=6)
    _check(torch, _run(torch, x, lens, 32, 8, kind), x, lens, 32, 8, kind)
    _check(torch, _run(torch, x, lens, 32, 8, kind, window=301), x, lens, 32, 8, kind, window=301)
    _check(torch, _run(torch, x, lens, 32, 8, kind, causal=False), x, lens, 32, 8, kind, causal=False)


@pytest.mark.parametrize("kind", KINDS)
def test_one_head_each_and_many_heads(cuda, kind):
    torch = cuda
    for hq, hk, n in ((20, 20, 260), (150, 1, 40), (35, 5, 130)):
        x = _rows(torch, kind, [n], hq, hk, seed=hq)
        _check(torch, _run(torch, x, [n], hq, hk, kind), x, [n], hq, hk, kind)


@pytest.mark.parametrize("kind", KINDS)
def test_without_row_begin_and_with_a_scale(cuda, kind):
    torch = cuda
    x = _rows(torch, kind, [201], 4, 1, seed=7)
    _check(torch, _run(torch, x, [201], 4, 1, kind, begin=None, scale=0.031), x, [201], 4, 1, kind, scale=0.031)


@pytest.mark.parametrize("kind", KINDS)
def test_scores_that_grow_along_the_sequence(cuda, kind):
    """The largest score moves with every block, so that the sums are brought along."""
    torch, n = cuda, 900
    x = _rows(torch, kind, [n], 2, 1, seed=8)
    x[:, :2] = x[:, :2].abs()
    ramp = torch.linspace(0.0, 3.0, n, device="cuda")[:, None]
    x[:, 2] = (x[:, 2].float().abs() * ramp).to(x.dtype)
    _check(torch, _run(torch, x, [n], 2, 1, kind), x, [n], 2, 1, kind)
    x[:, 2] = x[:, 2].flip(0)  # and falls, so that what follows is small beside it
    _check(torch, _run(torch, x, [n], 2, 1, kind), x, [n], 2, 1, kind)


@pytest.mark.parametrize("kind", KINDS)
def test_rows_of_no_sequence_and_empty_sequences(cuda, kind):
    torch, lens = cuda, [0, 70, 0, 0, 140, 0]
    x = _rows(torch, kind, lens, 4, 2, seed=9, pad=30)
    begin = _begin(torch, lens, offset=11)
    out = _run(torch, x, lens, 4, 2, kind, begin=begin)
    assert (out[:11] == 7).all() and (out[221:] == 7).all()
    _check(torch, out, x, lens, 4, 2, kind, at=11)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), "lowest"])
def test_masked_values_do_not_matter(cuda, kind, bad):
    """Tokens after a row, before its window, of the next sequence and of no sequence."""
    torch, lens = cuda, [150, 90]
    x = _rows(torch, kind, lens, 4, 2, seed=10, pad=40)
    clean = x.clone()
    bad = torch.finfo(x.dtype).min if bad == "lowest" else bad
    x[240:] = bad           # of no sequence
    x[100, 4:] = bad        # rows before token 100 do not see it
    x[150 + 3, 4:] = bad    # nor rows from 153 + 60 on
    for window in (0, 60):
        out = _run(torch, x, lens, 4, 2, kind, window=window)
        ref = _run(torch, clean, lens, 4, 2, kind, window=window)
        assert torch.equal(out[:100], ref[:100]) and torch.equal(out[150:153], ref[150:153])
        if window:
            assert torch.equal(out[100 + 60:150], ref[100 + 60:150]) and torch.equal(out[153 + 60:240], ref[153 + 60:240])


@pytest.mark.parametrize("kind", KINDS)
def test_values_that_are_not_finite_reach_the_rows_that_see_them(cuda, kind):
    torch, n = cuda, 300
    x = _rows(torch, kind, [n], 4, 2, seed=11)
    x[200, 6, 5] = float("inf")
    x[130, 7, 9] = float("nan")
    out = _run(torch, x, [n], 4, 2, kind)
    assert torch.isfinite(out[:130]).all()
    assert torch.isnan(out[130:, 2:, 9]).all() and torch.isfinite(out[:, 2:, :9]).all()
    # where the probability is not zero in fp32, the formula says infinity; far behind it may be zero times it
    assert not torch.isfinite(out[200:, :2, 5]).any() and torch.isfinite(out[:200, :2]).all()
    assert torch.isfinite(out[:, :2, 6:]).all()


def test_strides_streams_and_two_calls_at_once(cuda):
    torch, lens = cuda, [260, 31]
    x = _rows(torch, "bf16", lens, 4, 2, seed=12)
    want = _run(torch, x, lens, 4, 2, "bf16")
    wide = torch.full((291, 4 * 128 + 8), 3.0, dtype=torch.bfloat16, device="cuda")
    streams = [torch.cuda.Stream() for _ in range(4)]
    outs = [torch.empty_like(want) for _ in streams]
    torch.cuda.synchronize()
    for s, o in zip(streams, outs):
        with torch.cuda.stream(s):
            _run_on(torch, x, lens, o, s)
    _run_on(torch, x, lens, wide, None, output_stride=wide.shape[1])
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)
    assert torch.equal(wide[:, :512].reshape(-1, 4, 128), want) and (wide[:, 512:] == 3).all()


def _run_on(torch, x, lens, out, stream, **more):
    import qwanto_b200 as qb
    flat = x.view(x.shape[0], -1)
    qb.prompt_attention(flat, flat[:, 4 * 128:], flat[:, 6 * 128:], out, x.shape[0], 3, 4, 2, num_seqs=len(lens),
                        row_begin=_held(torch, lens), query_stride=1024, key_stride=1024, value_stride=1024,
                        stream=stream, **more)


_HELD = {}


def _held(torch, lens):
    """The same offsets for every stream: made before, not on one of them."""
    key = tuple(lens)
    if key not in _HELD:
        _HELD[key] = _begin(torch, lens)
        torch.cuda.synchronize()
    return _HELD[key]


def test_capture_and_replay_with_other_lengths(cuda):
    """The lengths are read on the device: a captured call serves other batches of as many rows."""
    torch = cuda
    lens, other = [200, 56], [17, 239]
    x = _rows(torch, "f16", lens, 4, 2, seed=13)
    begin, out = _begin(torch, lens), torch.empty((256, 4, 128), dtype=torch.float16, device="cuda")
    _run(torch, x, lens, 4, 2, "f16", out=out, begin=begin)
    graph = torch.cuda.CUDAGraph()
    import qwanto_b200 as qb
    flat = x.view(256, -1)
    with torch.cuda.graph(graph):
        qb.prompt_attention(flat, flat[:, 512:], flat[:, 768:], out, 256, 2, 4, 2, num_seqs=2, row_begin=begin,
                            query_stride=1024, key_stride=1024, value_stride=1024, stream=torch.cuda.current_stream())
    for n in (lens, other, [256, 0], [0, 100]):
        begin.copy_(_begin(torch, n))
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        _check(torch, out, x, n, 4, 2, "f16")


@pytest.mark.parametrize("kind", KINDS)
def test_same_bits_every_time(cuda, kind):
    torch, lens = cuda, [700, 41, 300]
    x = _rows(torch, kind, lens, 12, 2, seed=14)
    first = _run(torch, x, lens, 12, 2, kind)
    for _ in range(3):
        assert torch.equal(first, _run(torch, x, lens, 12, 2, kind))


def test_a_row_that_must_start_on_16_bytes(cuda):
    import qwanto_b200 as qb
    torch = cuda
    x = torch.zeros((8, 3 * 128 + 4), dtype=torch.bfloat16, device="cuda")
    out = torch.zeros((8, 128), dtype=torch.bfloat16, device="cuda")
    with pytest.raises(qb.QwnCudaError):
        qb.prompt_attention(x, x[:, 128:], x[:, 256:], out, 8, 3, 1, 1, query_stride=388, key_stride=388, value_stride=388)
