"""CPU tests around the 4-bit cache: refusals of the tensor-level functions and of the C ABI before any device work, frequencies of
the rotary positions, and the restatements that the GPU tests compare with."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from . import kv4_reference as R


@pytest.fixture(scope="module")
def kv4():
    from decdec_b200 import kv4 as m
    return m


@pytest.fixture(scope="module")
def capi():
    from decdec_b200 import capi as m
    return m


def half(*shape):
    return torch.zeros(shape, dtype=torch.float16)


def ints(*shape, dtype=torch.int32):
    return torch.zeros(shape, dtype=dtype)


def test_cache_shapes(kv4):
    assert tuple(kv4.empty_cache(3, 64, 8, 128, 128, device="cpu").shape) == (3, 8, 4 * 16 * 136)
    assert tuple(kv4.empty_cache(1, 16, 1, 64, 32, device="cpu").shape) == (1, 1, 16 * 80)
    for bad in ((3, 24, 8, 128, 128), (3, 0, 8, 128, 128), (3, 16, 8, 96, 32), (3, 16, 8, 64, 128), (3, 16, 8, 128, 16)):
        with pytest.raises(RuntimeError):
            kv4.empty_cache(*bad, device="cpu")


def test_tensor_refusals(kv4):
    cache = kv4.empty_cache(2, 16, 2, 128, 64, device="cpu")
    f = torch.ones(64, dtype=torch.float64)
    with pytest.raises(RuntimeError, match="must be on GPU"):
        kv4.rotary(half(1, 2, 128), None, ints(1), f)
    with pytest.raises(RuntimeError, match="shape"):
        kv4.rotary(half(2, 128), None, ints(1), f)
    with pytest.raises(RuntimeError, match="neighbours"):
        kv4.rotary(half(1, 128, 2).transpose(1, 2), None, ints(1), f)
    with pytest.raises(RuntimeError, match="Unsupported data type"):
        kv4.rotary(torch.zeros(1, 2, 128, dtype=torch.float64), None, ints(1), f)
    with pytest.raises(RuntimeError, match="both be half"):
        kv4.append(cache, torch.zeros(1, 2, 128), torch.zeros(1, 2, 128), ints(1), 64)
    with pytest.raises(RuntimeError, match="must be on GPU"):
        kv4.append(cache, half(1, 2, 128), half(1, 2, 128), ints(1), 64)
    with pytest.raises(RuntimeError, match="same shape"):
        kv4.append(cache, half(1, 2, 128), half(1, 2, 64), ints(1), 64)
    with pytest.raises(RuntimeError, match="dtype must be"):
        kv4.gather(cache, ints(1), 128, 64, torch.float32)
    with pytest.raises(RuntimeError, match="must be on GPU"):
        kv4.gather(cache, ints(1), 128, 64, torch.float16)
    with pytest.raises(RuntimeError, match="q must be half"):
        kv4.attention(torch.zeros(1, 2, 128), cache, ints(1, 1), ints(1), ints(2), 64)
    with pytest.raises(RuntimeError, match="must be on GPU"):
        kv4.attention(half(1, 2, 128), cache, ints(1, 1), ints(1), ints(2), 64)
    with pytest.raises(RuntimeError, match="must be on GPU"):
        kv4.plan(ints(1), ints(1), ints(1, 1), ints(1), ints(1), 16, 1)


def test_status_codes_without_gpu(capi):
    lib, H, B, F = capi.lib, capi.FP16, capi.BF16, capi.FP32

    def rotary(d=128, r=128, dtype=H, q=16, heads=1):
        return lib.decdec_rotary(q, 128, 128, heads, None, 0, 0, 0, 16, 128, 128, None, 0, 0, 16, 1, 16, 1, d, r, 0, 1.0, dtype, None)

    assert rotary(r=130) == -1 and rotary(r=3) == -1 and rotary(r=0) == -1 and rotary(dtype=7) == -1 and rotary(q=None) == -1
    assert b"null pointer" in lib.decdec_last_error()
    assert rotary(d=4096, r=2048) == -2
    assert rotary(heads=0) == 0                                               # nothing to turn

    def plan(page=16, cols=4, starts=16, tokens=1, requests=1):
        return lib.decdec_kv4_plan(16, 16, requests, 16, cols, cols, 16, 1, 16, page, tokens, 16, 16, starts, 16, 16, 16, None)

    assert plan(page=0) == -1 and plan(page=24) == -1 and plan(page=65552) == -1 and plan(starts=None) == -1
    assert plan(cols=1 << 28) == -1 and plan(tokens=1 << 31) == -1
    assert b"below 2^31" in lib.decdec_last_error()

    def append(d=128, g=128, page=16, dtype=H, cache=16, pages=1, heads=1, k=16, tokens=1):
        return lib.decdec_kv4_append(k, d, d, 16, d, d, 16, 1, tokens, cache, pages, page, heads, d, g, dtype, None)

    def gather(d=128, g=128, page=16, dtype=H, cache=16, pages=1, heads=1, out=16, tokens=1):
        return lib.decdec_kv4_gather(cache, pages, page, heads, d, g, 16, 1, tokens, out, 16, dtype, None)

    for call in (append, gather):
        assert call(d=96, g=32) == -2 and call(g=16) == -1 and call(d=64, g=128) == -1 and call(page=20) == -1 and call(dtype=F) == -1
        assert call(cache=None) == -1 and call(cache=8) == -1 and call(pages=0) == -1 and call(heads=0) == -1
        assert call(tokens=0) == 0 and call(tokens=1 << 31) == -2
    assert append(k=None) == -1 and gather(out=None) == -1 and gather(out=4) == -1

    n = C.c_size_t(0)

    def attention(d=128, g=128, heads=8, kv=2, page=16, dtype=B, rows=1, requests=1, cols=4, scale=0.1, cache=16, out=16, most=1, st=128):
        return lib.decdec_kv4_attention(16, 128, 128, out, st, 128, None, cache, 4, page, 16, cols, cols, 16, 16, requests, rows, heads, kv, d, g,
                                        most, scale, 0, 0, 16, 1 << 30, dtype, None)

    assert attention(d=96, g=32) == -2 and attention(g=256) == -1 and attention(heads=7) == -1 and attention(kv=0) == -1 and attention(dtype=F) == -1
    assert attention(page=8) == -1 and attention(cols=1 << 28) == -1 and attention(most=0) == -1
    for scale in (0.0, -1.0, math.inf, math.nan):
        assert attention(scale=scale) == -1
    assert b"positive" in lib.decdec_last_error()
    assert attention(rows=0) == 0
    assert attention(cache=8) == -1 and attention(out=4) == -1 and attention(st=130) == -1 and attention(out=None) == -1
    assert attention(rows=1 << 30) == -2
    assert lib.decdec_kv4_attention_workspace(1, 1, 8, 2, 128, 128, 1, H, None) == -1
    assert lib.decdec_kv4_attention_workspace(1, 1, 8, 3, 128, 128, 1, H, C.byref(n)) == -1


def test_rotary_frequencies(kv4):
    f, factor = kv4.rotary_frequencies(64, 10000.0, device="cpu")
    assert f.dtype == torch.float64 and factor == 1.0
    assert all(abs(f[i].item() - 10000.0 ** (-2 * i / 64)) <= 1e-15 for i in range(32))
    g, _ = kv4.rotary_frequencies(64, 10000.0, {"type": "linear", "factor": 4.0}, device="cpu")
    assert torch.equal(g, f / 4)
    s = {"type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0, "original_max_position_embeddings": 8192}
    g, _ = kv4.rotary_frequencies(128, 500000.0, s, device="cpu")
    for i in range(64):                                                       # the published rule, by wave lengths
        base = 500000.0 ** (-2 * i / 128)
        wave = 2 * math.pi / base
        if wave < 8192 / 4.0:
            want = base
        elif wave > 8192 / 1.0:
            want = base / 8
        else:
            smooth = (8192 / wave - 1.0) / (4.0 - 1.0)
            want = (1 - smooth) * base / 8 + smooth * base
        assert abs(g[i].item() - want) <= 1e-14 * want
    s = {"type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096}
    g, factor = kv4.rotary_frequencies(128, 10000.0, s, device="cpu")
    assert abs(factor - (0.1 * math.log(16.0) + 1)) < 1e-15
    f, _ = kv4.rotary_frequencies(128, 10000.0, device="cpu")
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(g[turns > 40], f[turns > 40]) and torch.allclose(g[turns < 0.8], f[turns < 0.8] / 16, rtol=1e-14)
    assert ((g <= f) & (g >= f / 16 * (1 - 1e-14))).all()
    for bad in ({"type": "dynamic", "factor": 2.0}, {"type": "linear", "factor": 0.5}, {"type": "llama3", "factor": 2.0, "low_freq_factor": 4.0,
                "high_freq_factor": 1.0, "original_max_position_embeddings": 8192}):
        with pytest.raises(RuntimeError):
            kv4.rotary_frequencies(64, 10000.0, bad, device="cpu")
    with pytest.raises(RuntimeError):
        kv4.rotary_frequencies(63, 10000.0, device="cpu")


@pytest.mark.parametrize("d,group", [(64, 32), (128, 128), (256, 64)])
def test_every_byte_of_a_cell_has_one_owner(d, group):
    """The restated format puts the words of 16 tokens side by side without gaps or overlaps."""
    g = torch.Generator().manual_seed(1)
    seen = np.zeros((16, R.cell_bytes(d, group)), dtype=bool)
    for r in range(16):
        x = torch.randn(1, d, generator=g).half()
        a, b = np.zeros((1, 1, R.cell_bytes(d, group)), np.uint8), np.full((1, 1, R.cell_bytes(d, group)), 255, np.uint8)
        R.write_row(a, r, x, x, group, 16)
        R.write_row(b, r, x, x, group, 16)
        seen[r] = (a == b)[0, 0]
    assert (seen.sum(0) == 1).all()


def test_restated_quantizer():
    x = torch.tensor([[0.0] * 31 + [15.0], [2.0] * 32, [float("nan")] + [1.0] * 31, [float("inf")] + [1.0] * 31], dtype=torch.bfloat16)
    x[0, 1:16] = torch.tensor([0.5, 1.5, 2.5, 3.5, 4.5, 5.5, 6.5, 7.5, 8.5, 9.5, 10.5, 11.5, 12.5, 13.5, 14.5])
    code, step, lo = R.quantize(x, 32)
    assert step[0, 0] == 1 and code[0, 1:16].tolist() == [0, 2, 2, 4, 4, 6, 6, 8, 8, 10, 10, 12, 12, 14, 14]       # ties to even
    assert step[1, 0] == 0 and lo[1, 0] == 2 and (code[1] == 0).all()
    assert math.isnan(lo[2, 0]) and math.isnan(lo[3, 0]) and step[2, 0] == 0
    assert torch.isnan(R.held(x, 32)[2:]).all()


@pytest.mark.parametrize("length", [65536, 131072])
def test_yarn_where_every_pair_turns_over_the_trained_length(kv4, length):
    """The ramp's upper end lies behind the last pair when the trained length is above 2 pi base: it is cut at the rotated elements, not at their pairs."""
    g, _ = kv4.rotary_frequencies(128, 10000.0, {"type": "yarn", "factor": 16.0, "original_max_position_embeddings": length}, device="cpu")
    # pairs with 32 turns and one turn over the length: 128 ln(length / (2 pi turns)) / (2 ln 10000) = 40.2 and 64.3, 45.03 and 69.1
    first, last = {65536: (40, 65), 131072: (45, 70)}[length]
    for i in range(64):
        slow = min(max((i - first) / (last - first), 0.0), 1.0)
        want = 10000.0 ** (-i / 64) * (1 - slow + slow / 16)
        assert abs(g[i].item() - want) <= 1e-13 * want, i
    assert g[63].item() / 10000.0 ** (-63 / 64) > {65536: 0.13, 131072: 0.32}[length]
