"""The serving operators without a GPU: what the C entry points and the Python functions refuse, and the oracle that the GPU tests compare
with (the plan, the order of the 4-bit codes, the quantisation) against properties that define it."""
import ctypes
import math
import os
import random
import subprocess
import sys

import numpy as np
import pytest
import torch

from oracle import serving_oracle as S

ONE = ctypes.c_void_p(4096)   # never dereferenced: validation comes first
TWO = ctypes.c_void_p(8192)


def refused(name, args, match):
    from clusterfusionplus_b200 import _lib
    assert getattr(_lib.lib, name)(*args) == -1
    assert match in _lib.last_error(), _lib.last_error()


def plan_args(**kw):
    a = dict(cached=ONE, new=ONE, batch=4, table=ONE, width=8, stride=8, free=ONE, n_free=16, count=ONE, count_out=TWO, page=16, kv_lens=TWO, qo=ONE,
             positions=ONE, slots=ONE, max_tokens=4, kv_indptr=ONE, kv_indices=ONE, max_rows=64, status=ONE, stream=None)
    return list((a | kw).values())


@pytest.mark.parametrize("kw,match", [
    (dict(cached=None), "null"), (dict(status=None), "null"), (dict(free=None), "null"), (dict(slots=None), "null"), (dict(kv_indices=None), "null"),
    (dict(batch=0), "batch"), (dict(batch=4097), "batch"), (dict(page=0), "page size"), (dict(width=0), "block table"), (dict(stride=7), "block table"),
    (dict(n_free=-1), "free list"), (dict(count_out=ONE), "alias"), (dict(kv_lens=ONE), "alias"), (dict(max_tokens=-1), "max_tokens"),
    (dict(max_rows=1 << 31), "max_rows"), (dict(kv_indices=ctypes.c_void_p(4100)), "aligned")])
def test_plan_refusals(kw, match):
    refused("cf_paged_kv_plan", plan_args(**kw), match)


@pytest.mark.parametrize("kw,match", [(dict(finished=None), "null"), (dict(batch=5000), "batch"), (dict(count_out=ONE), "alias"), (dict(page=1 << 20), "page size")])
def test_release_refusals(kw, match):
    a = dict(finished=ONE, kv_lens=ONE, batch=4, table=ONE, width=8, stride=8, free=ONE, n_free=16, count=ONE, count_out=TWO, page=16, status=ONE, stream=None)
    refused("cf_paged_kv_release", list((a | kw).values()), match)


@pytest.mark.parametrize("kw,match", [
    (dict(dim=132), "head_dim"), (dict(dim=12), "head_dim"), (dict(dim=8), "head_dim"), (dict(page=24), "page size"), (dict(page=0), "page size"), (dict(pages=0), "pages"),
    (dict(pages=1 << 27), "pages"), (dict(dtype=2), "dtype"), (dict(tokens=-1), "tokens"), (dict(key=None), "null"), (dict(kts=130), "stride"),
    (dict(key=ctypes.c_void_p(4098)), "aligned"), (dict(cache=ctypes.c_void_p(4104)), "16 bytes")])
def test_append_refusals(kw, match):
    a = dict(key=ONE, value=ONE, dtype=0, tokens=3, heads=2, dim=128, kts=256, khs=128, vts=256, vhs=128, slots=ONE, cache=ONE, pages=4, page=16, stream=None)
    refused("cf_kv4_append", list((a | kw).values()), match)


@pytest.mark.parametrize("kw,match", [(dict(dim=0), "head_dim"), (dict(dtype=5), "dtype"), (dict(key=None), "null"), (dict(value=ctypes.c_void_p(8)), "aligned"), (dict(heads=0), "heads")])
def test_read_refusals(kw, match):
    a = dict(cache=ONE, pages=4, page=16, heads=2, dim=128, slots=ONE, tokens=3, key=ONE, value=ONE, dtype=1, stream=None)
    refused("cf_kv4_read", list((a | kw).values()), match)


@pytest.mark.parametrize("kw,match", [
    (dict(dim=100), "head_dim"), (dict(heads=5), "query heads"), (dict(heads=2), "query heads"), (dict(rows=-1), "rows"), (dict(batch=0), "batch"), (dict(qo=None), "query rows"),
    (dict(max_q=0), "max_q_len"), (dict(width=0), "block table"), (dict(stride=3), "block table"), (dict(query=None), "null"), (dict(out=None), "null"),
    (dict(qts=1020), "strides"), (dict(query=ctypes.c_void_p(8)), "aligned"), (dict(dtype=2), "dtype"), (dict(page=17), "page size"),
    (dict(work=ONE, work_bytes=16, width=1 << 14, stride=1 << 14), "workspace"), (dict(work=ctypes.c_void_p(8), work_bytes=1 << 30, width=1 << 14, stride=1 << 14), "workspace")])
def test_attention_refusals(kw, match):
    a = dict(query=ONE, dtype=0, rows=3, heads=8, dim=128, qts=1024, qhs=128, cache=ONE, pages=4, page=16, kv_heads=4, table=ONE, width=8, stride=8, kv_lens=ONE, qo=ONE, batch=4,
             max_q=1, scale=0.1, work=None, work_bytes=0, out=ONE, stream=None)
    refused("cf_kv4_attention", list((a | kw).values()), match)


def test_attention_refuses_a_hint_beyond_any_call():
    from clusterfusionplus_b200._lib import lib
    a = [ONE, 0, 3, 8, 128, 1024, 128, ONE, 4, 16, 4, ONE, 8, 8, ONE, ONE, 4, 1 << 62, 0.1, None, 0, ctypes.c_void_p(1 << 20), None]
    refused("cf_kv4_attention", a, "max_q_len")
    assert lib.cf_kv4_attention_workspace(4, 8, 4, 128, 1 << 14, 1 << 62) == 0
    assert lib.cf_kv4_attention_workspace(4, 1 << 62, 1 << 61, 128, 1 << 14, 4) == 0


@pytest.mark.parametrize("at", [0, 256 * 7, 2 * 1024 * 2 + 2 * 1024 - 16])
@pytest.mark.parametrize("first", ["query", "out"])
def test_attention_refuses_an_output_over_the_queries(at, first):
    """3 rows of 8 heads of 128: 6144 bytes each; the other tensor starts inside the first."""
    base, shifted = ctypes.c_void_p(1 << 20), ctypes.c_void_p((1 << 20) + at)
    q, o = (base, shifted) if first == "query" else (shifted, base)
    refused("cf_kv4_attention", [q, 0, 3, 8, 128, 1024, 128, ONE, 4, 16, 4, ONE, 8, 8, ONE, ONE, 4, 1, 0.1, None, 0, o, None], "overlaps")


@pytest.mark.parametrize("kw,match", [
    (dict(dtype=3), "dtype"), (dict(rows=-1), "rows"), (dict(vocab=0), "vocabulary"), (dict(top=33), "top_k"), (dict(top=-1), "top_k"), (dict(vocab=4), "top_k"), (dict(bytes=2), "tokens"),
    (dict(logits=None), "null"), (dict(tops=None), "null"), (dict(logits=ctypes.c_void_p(4097)), "aligned")])
def test_logprobs_refusals(kw, match):
    a = dict(logits=ONE, dtype=0, rows=3, vocab=100, stride=100, tokens=ONE, bytes=8, top=5, lp=ONE, entropy=ONE, tops=ONE, ids=ONE, stream=None)
    refused("cf_token_logprobs", list((a | kw).values()), match)


def test_nothing_to_do_is_fine():
    from clusterfusionplus_b200 import _lib
    lib = _lib.lib
    assert lib.cf_kv4_append(None, None, 0, 0, 2, 128, 256, 128, 256, 128, None, None, 4, 16, None) == 0
    assert lib.cf_kv4_read(None, 4, 16, 2, 128, None, 0, None, None, 0, None) == 0
    assert lib.cf_kv4_attention(None, 0, 0, 8, 128, 1024, 128, None, 4, 16, 4, None, 8, 8, None, ONE, 4, 1, 0.1, None, 0, None, None) == 0
    assert lib.cf_token_logprobs(None, 0, 0, 100, 100, None, 8, 0, None, None, None, None, None) == 0


def test_cpu_tensors_are_rejected():
    """On a box without a GPU there is no current device; on one with a GPU the tensors are named."""
    import clusterfusion as cf
    i = torch.zeros(2, dtype=torch.int32)
    x = torch.zeros(2, 2, 64, dtype=torch.float16)
    cache = torch.zeros(2, 2, 16, 80, dtype=torch.uint8)
    for call in (lambda: cf.paged_kv_plan(i, i, torch.zeros(2, 4, dtype=torch.int32), i, i[:1], 16, 2), lambda: cf.kv4_append(x, x, i, cache), lambda: cf.kv4_read(cache, i, 64),
                 lambda: cf.kv4_attention(x, cache, torch.zeros(2, 4, dtype=torch.int32), i), lambda: cf.token_logprobs(x[0], i),
                 lambda: cf.paged_kv_release(i, i, torch.zeros(2, 4, dtype=torch.int32), i, i[:1], 16)):
        with pytest.raises((RuntimeError, AssertionError)):
            call()
    with pytest.raises(RuntimeError, match="multiple of"):
        cf.kv4_cache(2, 2, 24, 128, device="cpu")
    assert cf.kv4_cache(2, 3, 32, 80, device="cpu").shape == (2, 3, 32, 120)


def test_binding_reports_what_is_wrong():
    """The compiled checks: messages with numbers and shapes in them arrive as Python exceptions."""
    from clusterfusionplus_b200 import serving
    x, i = torch.zeros(2, 2, 64, dtype=torch.float16), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="kv4_attention: 9 arguments, got 2"):
        serving._call.attention(x, i)
    with pytest.raises(RuntimeError, match="key: expected a torch.Tensor"):
        serving.kv4_append(None, x, i, x)
    with pytest.raises(RuntimeError, match="logits: expected a CUDA tensor, got cpu"):
        serving.token_logprobs(x[0], i)


# ------------------------------------------------------------------------------------------------------------- oracle
@pytest.mark.parametrize("D", [16, 32, 64, 80, 96, 128])
def test_every_nibble_of_a_tile_has_one_owner(D):
    """Codes and parameters fill a tile without overlap, and the codes of four dims are one aligned 16-bit half."""
    G = S.groups(D)
    seen = {}
    for v in range(2):
        for t in range(16):
            for d in range(32 * G):
                byte, shift = S.nibble(D, t, d, v)
                assert (byte, shift) not in seen and byte < 512 * G
                seen[byte, shift] = 1
                base = S.nibble(D, t, d // 4 * 4, v)[0]
                assert base % 2 == 0 and (byte, shift) == (base + d % 4 // 2, 4 * (d % 2))
    params = {S.param(D, t, w, g) for t in range(16) for w in range(4) for g in range(G)}
    assert len(seen) == 2 * 16 * 32 * G and params == set(range(512 * G, 640 * G, 2))


@pytest.mark.parametrize("D", [16, 80, 128])
def test_quantisation_is_within_half_a_step(D):
    rng = np.random.RandomState(D)
    x = rng.standard_normal((50, D)).astype(np.float16).astype(np.float32) * np.float32(2.0)
    c, s, m = S.quantise(x)
    g = np.arange(D) // 32
    back = c * s.astype(np.float64)[:, g] + m.astype(np.float64)[:, g]
    # half a step; the top code stands up to 15 half-ulps of the scale below the maximum
    assert (np.abs(back - x) <= s.astype(np.float64)[:, g] * (0.5 + 15 * 2.0 ** -11 + 1e-6)).all()


def test_quantisation_of_constant_and_broken_groups():
    x = np.full((1, 64), 1.5, np.float32)
    x[0, 40] = np.nan
    c, s, m = S.quantise(x)
    assert s[0, 0] == 0 and m[0, 0] == 1.5 and (c == 0).all() and np.isnan(s[0, 1])
    for bad in (np.inf, -np.inf):
        assert np.isnan(S.quantise(np.array([[bad] + [0.0] * 31], np.float32))[1]).all()
    c, s, m = S.quantise(np.array([[1e38, -1e38] + [0.0] * 30], np.float32))   # bf16 reaches further than fp16
    assert m[0, 0] == -65504 and c[0, 0] == 15 and c[0, 1] == 0


def test_store_and_unpack_are_inverse():
    rng = np.random.RandomState(3)
    cache = rng.randint(0, 256, (3, 2, 32, 120)).astype(np.uint8)
    cache.reshape(3, 2, 2, 1920)[..., 1536:] = 0
    before = cache.copy()
    key, value = rng.standard_normal((2, 2, 80)).astype(np.float16).astype(np.float32)
    S.store(cache, 2 * 32 + 21, key, value)
    k, v = S.unpack(cache, 80)
    k0, v0 = S.unpack(before, 80)
    for got, old, x in ((k, k0, key), (v, v0, value)):
        c, s, m = S.quantise(x)
        g = np.arange(80) // 32
        assert np.array_equal(got[2, :, 21].numpy(), c * s.astype(np.float64)[:, g] + m.astype(np.float64)[:, g])
        got[2, :, 21] = old[2, :, 21]
        assert torch.equal(got, old)


def test_plan_of_the_oracle():
    got = S.plan([16, 0, 5], [1, 0, 12], [[7, -1], [-1, -1], [3, -1]], [9, 4, 8], 3, 16, 15, 40)
    assert got["status"] == 0 and got["table"] == [[7, 8], [-1, -1], [3, 4]] and got["free_count"] == 1
    assert got["qo_indptr"] == [0, 1, 1, 13] and got["positions"][:3] == [16, 5, 6] and got["slot_map"][0] == 8 * 16
    assert got["slot_map"][1:13] == [53 + i for i in range(11)] + [64] and got["slot_map"][13:] == [-1, -1]
    assert got["kv_indptr"] == [0, 17, 17, 34] and got["kv_indices"][:17] == list(range(112, 128)) + [128] and got["kv_indices"][34:] == [-1] * 6
    full = S.plan([16, 0, 5], [1, 0, 12], [[7, -1], [-1, -1], [3, -1]], [9], 1, 16, 12, 3)
    assert full["status"] == 1 + 4 + 8 and full["table"][0] == [7, -1] and full["kv_lens"] == [16, 0, 5] and full["free_count"] == 1


@pytest.mark.parametrize("count", [4, 90, -1])
def test_plan_of_the_oracle_refuses_a_count_beyond_the_list(count):
    got = S.plan([0], [0], [[-1]], [9, 8, 7], count, 16, 4, 0)
    assert got["status"] == 1 and got["free_count"] == count and got["table"] == [[-1]]


def test_logprobs_of_the_oracle():
    x = torch.tensor([[0.0, math.log(3.0), -math.inf, math.log(3.0)]])
    lp, h, tl, ti = S.logprobs(x, [1], 3)
    tol = 4 * 2.0 ** -24 * math.log(3.0)    # the logit log 3 is held in fp32: off by at most 2^-24 log 3, which p log p and log p pass on at most doubled
    assert abs(lp[0] - math.log(3 / 7)) < tol and ti.tolist() == [[1, 3, 0]]
    assert abs(h[0] - (-(6 / 7) * math.log(3 / 7) - (1 / 7) * math.log(1 / 7))) < tol
    assert S.logprobs(x, [2], 0)[0][0] == -math.inf and S.logprobs(x, [9], 0)[0][0] == -math.inf


def test_random_plans_keep_every_page_once():
    rng = random.Random(5)
    for _ in range(20):
        B, page = rng.randint(1, 9), rng.choice([1, 3, 16])
        lens = [rng.randint(0, 40) for _ in range(B)]
        new = [rng.randint(0, 20) for _ in range(B)]
        ids = list(range(400))
        rng.shuffle(ids)
        table = [[-1] * 64 for _ in range(B)]
        for b, n in enumerate(lens):
            for i in range(-(-n // page)):
                table[b][i] = ids.pop()
        got = S.plan(lens, new, table, ids, len(ids), page, 200, 0)
        used = [e for r in got["table"] for e in r if e >= 0]
        assert got["status"] == 0 and sorted(used + ids[:got["free_count"]]) == list(range(400))


@pytest.mark.parametrize("lo,hi", [(0.0, 65504.0), (-65504.0, 65504.0), (-1.0, 65504.0), (-1e38, 1e38), (-30000.0, 65504.0), (60000.0, 65504.0)])
def test_quantised_values_stay_within_fp16(lo, hi):
    """m + 15 s is an fp16 number where s would round it beyond (0 .. 65504: s = 4368, 15 x 4368 = 65520), and no further off than half a step."""
    x = np.linspace(lo, hi, 32).astype(np.float32)
    c, s, m = S.quantise(x[None])
    back = c[0] * s[0].astype(np.float64) + m[0].astype(np.float64)
    assert np.abs(back).max() <= 65504 and c[0, 0] == 0 and c[0, -1] == 15
    held = np.clip(x.astype(np.float64), -65504, 65504)
    assert (np.abs(back - held) <= s.astype(np.float64)[0] * (0.5 + 15 * 2.0 ** -10)).all()


def test_another_torch_does_not_keep_the_package_from_loading():
    """Only the serving calls need the module that is built for one torch: they say so, everything else works."""
    code = """
import torch
torch.__version__ = "99.0.0a0+other"
import clusterfusionplus_b200 as cf
assert cf.kv4_cache(1, 1, 16, 64, device="cpu").shape == (1, 1, 16, 80)
from clusterfusionplus_b200.api import model_dims
try:
    cf.kv4_append(None, None, None, None)
except ImportError as e:
    assert "was built for torch" in str(e) and "99.0.0a0+other" in str(e), e
    print("said so")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0 and "said so" in r.stdout, r.stdout + r.stderr


def test_a_build_for_another_torch_is_out_of_date(monkeypatch):
    from clusterfusionplus_b200 import build
    assert build.torch_version() == str(torch.__version__)
    assert not build._binding_stale()
    monkeypatch.setattr(build, "torch_version", lambda: "99.0.0")
    assert build._binding_stale() and not build.up_to_date()


@pytest.mark.parametrize("batch,tokens,q,line", [
    (64, 8192, 1, True), (1, 16384, 1, True), (4, 16384, 1, True), (32, 4096, 1, False), (16, 1000, 8, False), (20, 4096, 1, False), (20, 4112, 1, True),   # up to 8 rows: 592 CTAs at once
    (1, 16384, 12, True), (2, 16384, 12, True), (4, 16384, 12, False), (32, 8192, 12, False), (32, 16384, 12, True), (16, 16384, 12, True), (64, 16384, 12, False)])   # 9 to 16: 296
def test_the_line_is_taken_where_it_was_measured_faster(batch, tokens, q, line):
    """8 cached heads of 128, one query head each: room for half as many CTAs with 9 to 16 query rows moves the bounds."""
    from clusterfusionplus_b200._lib import lib
    assert (lib.cf_kv4_attention_workspace(batch, 8, 8, 128, tokens, q) > 0) == line


def test_the_plan_s_status_bits_have_names():
    """Those of the C header, in the package and its drop-in name."""
    import re

    import clusterfusion
    import clusterfusionplus_b200 as cf
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "clusterfusion_b200.h")).read()
    bits = re.findall(r"#define (CF_PLAN_[A-Z_]+) (\d+)", header)
    assert len(bits) == 6 and all(getattr(cf, n) == int(v) == getattr(clusterfusion, n) for n, v in bits)
