"""The paged 8-bit decode cache without a GPU: the C ABI's argument checks, the rotary
frequencies, and the refusal to run on host tensors."""

import ctypes
import math
import subprocess

import pytest
import torch

from submission_folder_b200 import _lib, ops
from submission_folder_b200.cache import PagedKVCache
from submission_folder_b200.rotary import rotary_frequencies

P = 4096   # a pointer that is never followed: every call here is refused first


def _cache(**over):
    a = dict(k=P, v=P, k_scale=P, v_scale=P, k_block_stride=4096, k_head_stride=2048, k_tok_stride=128, v_block_stride=4096,
             v_head_stride=2048, v_tok_stride=128, num_blocks=4, num_kv_heads=2, block_size=16, head_dim=128, format=0)
    a.update(over)
    return _lib.Cache(**a)


@pytest.mark.parametrize("over,code", [
    (dict(k=None), -1), (dict(v_scale=None), -1), (dict(format=2), -2), (dict(head_dim=96), -3), (dict(block_size=24), -3),
    (dict(num_blocks=0), -1), (dict(num_kv_heads=0), -1), (dict(num_kv_heads=40000), -1), (dict(k=P + 8), -1), (dict(k_scale=P + 2), -1),
    (dict(v_tok_stride=120), -1), (dict(k_head_stride=2056), -1)])
def test_bad_caches_are_refused(over, code):
    lib, c = _lib.load(), _cache(**over)
    assert lib.ckv_cache_read(ctypes.byref(c), P, P, 0, P, 3, None) == code
    assert lib.ckv_cache_write(ctypes.byref(c), P, 256, 128, P, 256, 128, 0, P, 3, None) == code
    a = _lib.AttentionArgs(q=P, q_tok_stride=1024, q_head_stride=128, out=P, out_tok_stride=1024, out_head_stride=128, tables=P,
                           table_stride=4, table_width=4, lens=P, requests=1, tokens=1, max_q=1, q_heads=8, scale=1.0)
    assert lib.ckv_cache_attention(ctypes.byref(c), ctypes.byref(a), P, 1 << 30, None) == code
    assert lib.ckv_last_error_string()


def test_bad_rows_are_refused():
    lib, c = _lib.load(), _cache()
    ref = ctypes.byref(c)
    assert lib.ckv_cache_write(ref, P, 256, 128, P, 256, 128, 7, P, 3, None) == -2       # dtype
    assert lib.ckv_cache_write(ref, P, 256, 128, P, 256, 128, 0, None, 3, None) == -1    # no slots
    assert lib.ckv_cache_write(ref, P, 256, 128, P, 256, 128, 0, P, -1, None) == -1
    assert lib.ckv_cache_write(ref, P + 2, 256, 128, P, 256, 128, 0, P, 3, None) == -1   # alignment
    assert lib.ckv_cache_write(ref, P, 250, 128, P, 256, 128, 0, P, 3, None) == -1
    assert lib.ckv_cache_read(ref, P, None, 0, P, 3, None) == -1
    assert lib.ckv_cache_read(ref, P, P, 0, P + 4, 3, None) == -1                          # slots' alignment
    assert lib.ckv_cache_write(ref, None, 0, 0, None, 0, 0, 0, None, 0, None) == 0       # nothing to write
    assert lib.ckv_cache_read(None, P, P, 0, P, 3, None) == -1


@pytest.mark.parametrize("over,code", [
    (dict(q=None), -1), (dict(tables=None), -1), (dict(lens=None), -1), (dict(dtype=5), -2), (dict(q=P + 4), -1),
    (dict(out_tok_stride=1020), -1), (dict(q_heads=7), -1), (dict(max_q=0), -1), (dict(table_width=0), -1),
    (dict(table_stride=3), -1), (dict(lens=P + 2), -1), (dict(requests=1 << 30, tokens=1 << 30, table_width=4096, table_stride=4096), -3),
    (dict(tokens=2), -1), (dict(requests=-1), -1), (dict(cu=P, max_q=1 << 20), -3)])
def test_bad_attention_is_refused(over, code):
    lib, c = _lib.load(), _cache()
    a = dict(q=P, q_tok_stride=1024, q_head_stride=128, out=P, out_tok_stride=1024, out_head_stride=128, tables=P, table_stride=4,
             table_width=4, lens=P, requests=1, tokens=1, max_q=1, q_heads=8, scale=1.0)
    a.update(over)
    s = _lib.AttentionArgs(**a)
    assert lib.ckv_cache_attention(ctypes.byref(c), ctypes.byref(s), P, 1 << 40, None) == code


def test_attention_workspace_is_checked():
    lib, c = _lib.load(), _cache()
    a = _lib.AttentionArgs(q=P, q_tok_stride=1024, q_head_stride=128, out=P, out_tok_stride=1024, out_head_stride=128, tables=P,
                           table_stride=4, table_width=4, lens=P, requests=1, tokens=1, max_q=1, q_heads=8, scale=1.0)
    need = ctypes.c_size_t()
    assert lib.ckv_cache_attention_workspace(128, 1, 8, 2, ctypes.byref(need)) == 0 and need.value > 0
    for ws, size in ((None, need.value), (P + 64, need.value), (P, need.value - 1)):
        assert lib.ckv_cache_attention(ctypes.byref(c), ctypes.byref(a), ws, size, None) == -4
    assert lib.ckv_cache_attention_workspace(80, 1, 8, 2, ctypes.byref(need)) == -3
    assert lib.ckv_cache_attention_workspace(128, 1, 7, 2, ctypes.byref(need)) == -1
    assert lib.ckv_cache_attention_workspace(128, 1, 8, 2, None) == -1


@pytest.mark.parametrize("over", [dict(lens=None), dict(out_slots=None), dict(out_granted=None), dict(work=None, total=4096), dict(requests=0), dict(requests=8193),
                                  dict(total=-1), dict(table_width=0), dict(table_stride=1), dict(block_size=0),
                                  dict(free_capacity=-1), dict(lens=P + 2), dict(out_slots=P + 4)])
def test_bad_table_steps_are_refused(over):
    a = dict(lens=P, new_tokens=P, tables=P, table_stride=4, table_width=4, free_list=P, free_capacity=8, free_count=P,
             block_size=16, requests=2, total=2, out_lens=P, out_free_count=P, out_cu=P, out_slots=P, out_positions=P,
             out_granted=P, work=P)
    a.update(over)
    s = _lib.TableStep(**a)
    assert _lib.load().ckv_block_tables(ctypes.byref(s), None) == -1


def test_tables_of_more_blocks_than_32_bits_count_are_refused():
    s = _lib.TableStep(lens=P, new_tokens=P, tables=P, table_stride=1 << 20, table_width=1 << 20, free_list=P, free_capacity=8,
                       free_count=P, block_size=16, requests=2048, total=2, out_lens=P, out_free_count=P, out_cu=P, out_slots=P,
                       out_positions=P, out_granted=P, work=P)
    assert _lib.load().ckv_block_tables(ctypes.byref(s), None) == -3


def test_slots_past_a_row_are_refused():
    c = PagedKVCache(1, 8, 2, 60, 2, 64, 16, device="cpu")
    assert c.slots(1, 64).tolist() == [i % 16 for i in range(64)]       # a table of zeros
    for tokens in (65, -1):
        with pytest.raises(ValueError, match="at most 64"):
            c.slots(1, tokens)


@pytest.mark.parametrize("over,code", [(dict(q=None), -1), (dict(k_heads=1), -1), (dict(dtype=3), -2), (dict(rotary_dim=0), -1),
                                       (dict(rotary_dim=7), -1), (dict(rotary_dim=66), -1), (dict(tokens=-1), -1),
                                       (dict(q_heads=0), -1), (dict(head_dim=2048, rotary_dim=64), -1), (dict(positions=P + 4), -1),
                                       (dict(q=P + 1), -1), (dict(tokens=0), 0)])
def test_bad_rotary_is_refused(over, code):
    a = dict(q=P, q_tok_stride=64, q_head_stride=64, out_q=P, out_q_tok_stride=64, out_q_head_stride=64, positions=P, inv_freq=P,
             factor=1.0, tokens=2, q_heads=1, k_heads=0, head_dim=64, rotary_dim=64, dtype=0)
    a.update(over)
    s = _lib.RotaryArgs(**a)
    assert _lib.load().ckv_rotary(ctypes.byref(s), None) == code


def test_host_tensors_are_refused():
    """The kernels never run on the CPU."""
    x, i = torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int32)
    c = PagedKVCache(1, 4, 2, 32, 2, 64, 16, device="cpu")
    for call in (lambda: ops.rotary(x, None, i.long(), rotary_frequencies(64)[0]),
                 lambda: ops.cache_write(x, x, *c.layer(0), i.long()), lambda: ops.cache_read(*c.layer(0), i.long()),
                 lambda: ops.cache_attention(x, *c.layer(0), c.tables, c.lens), lambda: c.step(i)):
        with pytest.raises(RuntimeError):
            call()


@pytest.mark.parametrize("over", [dict(num_layers=0), dict(block_size=48), dict(head_dim=80), dict(dtype=torch.uint8),
                                  dict(max_tokens=0)])
def test_bad_paged_caches_are_refused(over):
    a = dict(num_layers=1, num_blocks=4, max_requests=2, max_tokens=32, num_key_value_heads=2, head_dim=64, block_size=16, device="cpu")
    with pytest.raises(ValueError):
        PagedKVCache(**{**a, **over})


def test_rotary_frequencies():
    f, factor = rotary_frequencies(128)
    assert f.dtype == torch.float64 and factor == 1.0 and f[0] == 1.0
    assert torch.allclose(f, torch.tensor([10000.0 ** (-2 * i / 128) for i in range(64)], dtype=torch.float64), rtol=1e-14)
    assert torch.equal(rotary_frequencies(64, scaling=dict(type="linear", factor=4.0))[0], rotary_frequencies(64)[0] / 4)
    # dynamic: unchanged up to the original length; at twice it the slowest pair turns as far as before
    s = dict(rope_type="dynamic", factor=1.0, original_max_position_embeddings=2048)
    assert torch.equal(rotary_frequencies(64, scaling=s, seq_len=100)[0], rotary_frequencies(64)[0])
    slow = rotary_frequencies(64, scaling=s, seq_len=4096)[0][-1] * 4096
    assert math.isclose(float(slow), float(rotary_frequencies(64)[0][-1]) * 2048, rel_tol=1e-12)
    # llama3: fast pairs stay, slow pairs are divided, the blend lies between
    s = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0, original_max_position_embeddings=8192)
    plain, got = rotary_frequencies(128, 500000.0)[0], rotary_frequencies(128, 500000.0, s)[0]
    wave = 2 * math.pi / plain
    assert torch.equal(got[wave < 2048], plain[wave < 2048]) and torch.allclose(got[wave > 8192], plain[wave > 8192] / 8, rtol=1e-15)
    mid = (wave > 2048) & (wave < 8192)
    smooth = (8192 / wave - 1.0) / 3.0
    assert mid.any() and torch.allclose(got[mid], ((1 - smooth) * plain / 8 + smooth * plain)[mid], rtol=1e-12)
    # yarn: ends as above, and the attention factor
    s = dict(rope_type="yarn", factor=16.0, original_max_position_embeddings=4096)
    got, factor = rotary_frequencies(128, 10000.0, s)
    plain = rotary_frequencies(128)[0]
    assert got[0] == plain[0] and math.isclose(float(got[-1]), float(plain[-1]) / 16, rel_tol=1e-12)
    assert math.isclose(factor, 0.1 * math.log(16.0) + 1.0) and torch.all(got <= plain) and torch.all(got >= plain / 16)
    assert rotary_frequencies(128, 10000.0, dict(s, attention_factor=1.0))[1] == 1.0
    for bad in (dict(rope_type="other", factor=2.0), dict(rope_type="linear", factor=0.5)):
        with pytest.raises(ValueError):
            rotary_frequencies(64, scaling=bad)
    for dim in (0, 3):
        with pytest.raises(ValueError):
            rotary_frequencies(dim)


def _yarn(dim, base, s):
    """YaRN's frequencies pair by pair, in Python floats."""
    by, n = s["factor"], s["original_max_position_embeddings"]
    where = [dim * math.log(n / (2 * math.pi * t)) / (2 * math.log(base)) for t in (s.get("beta_fast", 32), s.get("beta_slow", 1))]
    if s.get("truncate", True):
        where = [math.floor(where[0]), math.ceil(where[1])]
    lo, hi = max(where[0], 0), min(where[1], dim - 1)
    out = []
    for i in range(dim // 2):
        f = base ** (-2 * i / dim)
        stretch = min(max((i - lo) / (hi - lo), 0.0), 1.0)
        out.append(f * (1 - stretch) + f / by * stretch)
    return torch.tensor(out, dtype=torch.float64)


@pytest.mark.parametrize("dim,base,extra", [
    (64, 150000.0, dict(factor=32.0, beta_fast=32.0, beta_slow=1.0, truncate=False)), (64, 150000.0, dict(factor=32.0, truncate=True)),
    (128, 10000.0, dict(factor=40.0)), (64, 10000.0, dict(factor=40.0, beta_fast=32, beta_slow=1, mscale=1.0, mscale_all_dim=1.0)),
    (64, 10000.0, dict(factor=40.0, mscale=0.707, mscale_all_dim=1.0)), (64, 10000.0, dict(factor=4.0, mscale=None, mscale_all_dim=0))])
def test_yarn_dictionaries(dim, base, extra):
    """Each key of a config's dictionary has its effect: the ramp between fractional or whole pairs, and
    the factor on cosine and sine."""
    s = dict(rope_type="yarn", original_max_position_embeddings=4096, **extra)
    got, factor = rotary_frequencies(dim, base, s)
    assert torch.allclose(got, _yarn(dim, base, s), rtol=1e-12, atol=0)
    m = lambda x: 0.1 * x * math.log(extra["factor"]) + 1.0   # noqa: E731
    want = m(extra["mscale"]) / m(extra["mscale_all_dim"]) if extra.get("mscale") else m(1.0)
    assert math.isclose(factor, want, rel_tol=1e-14)


def test_rope_scaling_keys_that_would_be_lost_are_refused():
    yarn = dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=4096)
    for bad in (dict(mscale=0.7), dict(mscale_all_dim=1.0), dict(short_factor=[1.0]), dict(beta=32.0),
                dict(rope_theta=500000.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(64, scaling={**yarn, **bad})
    same = rotary_frequencies(64, scaling={**yarn, "rope_theta": 10000, "finetuned": True, "mrope_section": [16, 24, 24], "partial_rotary_factor": 0.5, "beta_fast": None})
    assert torch.equal(same[0], rotary_frequencies(64, scaling=yarn)[0])


def test_rows_that_overlap_are_refused():
    """Written rows that share memory: a race on the device."""
    lib = _lib.load()
    write = lambda **o: lib.ckv_cache_write(ctypes.byref(_cache(k=P, v=2 * P, k_scale=3 * P, v_scale=4 * P, **o)), P, 256, 128, P,  # noqa: E731
                                            256, 128, 0, P, 3, None)
    for over in (dict(k_block_stride=0), dict(v_block_stride=0), dict(v_head_stride=0), dict(k_tok_stride=0), dict(k_tok_stride=64),
                 dict(k_block_stride=2048), dict(v_tok_stride=256, v_head_stride=128, v_block_stride=2048)):
        assert write(**over) == -1 and b"overlap" in lib.ckv_last_error_string(), over
    for same in (dict(v=P), dict(v_scale=3 * P)):
        c = _cache(**{**dict(k=P, v=2 * P, k_scale=3 * P, v_scale=4 * P), **same})
        assert lib.ckv_cache_write(ctypes.byref(c), P, 256, 128, P, 256, 128, 0, P, 3, None) == -1
    a = dict(q=P, q_tok_stride=1024, q_head_stride=128, out=P, out_tok_stride=1024, out_head_stride=128, tables=P, table_stride=4,
             table_width=4, lens=P, requests=3, tokens=3, max_q=1, q_heads=8, scale=1.0)
    for over in (dict(out_tok_stride=0), dict(out_head_stride=0), dict(out_tok_stride=128), dict(out_head_stride=64)):
        s = _lib.AttentionArgs(**{**a, **over})
        assert lib.ckv_cache_attention(ctypes.byref(_cache()), ctypes.byref(s), P, 1 << 40, None) == -1
        assert b"overlap" in lib.ckv_last_error_string(), over
    a = dict(q=P, q_tok_stride=128, q_head_stride=64, out_q=P, out_q_tok_stride=128, out_q_head_stride=64, positions=P, inv_freq=P, k=P,
             k_tok_stride=64, k_head_stride=64, out_k=2 * P, out_k_tok_stride=64, out_k_head_stride=64, factor=1.0, tokens=2, q_heads=2,
             k_heads=1, head_dim=64, rotary_dim=64, dtype=0)
    for over in (dict(out_q_tok_stride=0), dict(out_q_head_stride=32), dict(out_k_tok_stride=32), dict(out_k=P)):
        s = _lib.RotaryArgs(**{**a, **over})
        assert lib.ckv_rotary(ctypes.byref(s), None) == -1 and b"overlap" in lib.ckv_last_error_string(), over


def test_the_library_builds_without_torch(monkeypatch):
    """libckv.so and the C ABI need neither Python's headers nor torch's: plain make does not ask for them, and the
    build goes on without the module that does."""
    from submission_folder_b200 import build as b
    dry = subprocess.run(["make", "-n", "-B", "-C", b.CSRC, "PYTHON=false"], capture_output=True, text=True, check=True).stdout
    assert "libckv.so" in dry and "ckv_torch" not in dry
    assert "ckv_torch.cpp" in subprocess.run(["make", "-n", "-B", "-C", b.CSRC, "torch"], capture_output=True, text=True, check=True).stdout
    assert b.torch_headers()
    calls = []
    monkeypatch.setattr(b, "_make", lambda target, verbose: calls.append(target))
    assert b.build().endswith("libckv.so") and calls == ["../libckv.so", "torch"]
    calls.clear()
    monkeypatch.setattr(b.sysconfig, "get_paths", lambda: {"include": "/nonexistent"})
    assert b.build().endswith("libckv.so") and calls == ["../libckv.so"]
