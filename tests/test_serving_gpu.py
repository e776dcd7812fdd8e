"""The serving operators on the GPU against oracle/serving_oracle.py (lists, 64-bit numbers), at the sizes, masks, strides and orders where they can
go wrong, and all of them together as a server's step uses them.

Tolerances.  u = finfo(dtype).eps / 2 is the relative error of a rounding.
 - lists, codes, parameters and untouched bytes: equal.
 - values read back: one rounding of the 32-bit value, u |v| (plus fp32's 2^-24 |v| and, for results below fp16's normal range, half its
   smallest step 2^-25).
 - attention: kernels may round probabilities, keys and values to fp16 once each (2^-11 relative) and the result once (u).  Rounded keys move a
   score by at most 2^-11 scale sum |q k| =: e, so a probability by the factor exp(2 e) at most; with V the largest |value| the
   result is off by at most (2 e + 2^-11 + 2^-11) V + u |o|, to which 2^-16 V is added for fp32 sums (128 products and up to 2^9
   partial sums of at most 2^-24 each) and 2^-22 for exp2.  Beside this bound for each element the whole result has to be nearer: roundings
   are independent, and over a head's 32 or more elements their root mean square is below a third of the bound; rel-L2 <= 1e-3 for fp16 results, 2.5e-3
   for bf16 (a uniform rounding error of at most 2^-8 has the root mean square 2^-8 / sqrt(3) = 2.3e-3 at worst).
 - log probabilities: x - m and its product with log2(e) round three times in fp32, ex2 is good to 2^-22, a sum over n terms adds in runs of at most
   n / 512 terms and trees: (n / 512 + 24) 2^-24 + 2^-22 relative on z and w; so 2 (n / 512 + 24 + 4) 2^-24 times max(1, |log p|, entropy's terms <= 12)."""
import math
import os
import random

import numpy as np
import pytest
import torch

from oracle import serving_oracle as S

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.fixture(autouse=True)
def clean_status(cuda_device):
    import clusterfusionplus_b200 as cf
    yield
    torch.cuda.synchronize()
    assert cf.device_status() == 0


# --------------------------------------------------------------------------------------------------------------- plan
def plan_case(rng, B, page, width, most_len, most_new, spare=7):
    lens = [rng.choice([0, rng.randint(0, most_len)]) for _ in range(B)]
    new = [rng.choice([0, 1, rng.randint(0, most_new)]) for _ in range(B)]
    pool = sum(-(-(a + b) // page) for a, b in zip(lens, new)) + spare
    ids = list(range(pool))
    rng.shuffle(ids)
    table = [[-1] * width for _ in range(B)]
    for b, n in enumerate(lens):
        for i in range(-(-n // page)):
            table[b][i] = ids.pop()
    return lens, new, table, ids


def check_plan(lens, new, table, free, count, page, max_tokens, max_rows, strided=False):
    import clusterfusionplus_b200 as cf
    want = S.plan(lens, new, table, free, count, page, max_tokens, max_rows)
    t = ints(table)
    if strided:
        wide = torch.full((len(table), t.shape[1] + 5), -77, dtype=torch.int32, device=DEV)
        wide[:, :t.shape[1]] = t
        t = wide[:, :t.shape[1]]
    p = cf.paged_kv_plan(ints(lens), ints(new), t, ints(free), ints([count]), page, max_tokens, max_rows)
    assert int(p.status) == want["status"]
    for name in ("kv_lens", "qo_indptr", "positions", "slot_map", "kv_indptr", "kv_indices"):
        assert getattr(p, name).tolist() == want[name], name
    assert int(p.free_count) == want["free_count"] and t.tolist() == want["table"]
    assert p.positions.dtype == torch.int64
    if strided:
        assert (wide[:, -5:] == -77).all()
    return p


@pytest.mark.parametrize("B,page,most_len,most_new", [(1, 16, 100, 1), (1, 1, 5, 3), (2, 16, 0, 40), (16, 16, 500, 1), (33, 64, 900, 70), (255, 32, 300, 9), (256, 128, 2000, 1),
                                                      (257, 16, 90, 30), (1025, 16, 60, 4), (4096, 16, 20, 2)])
@pytest.mark.parametrize("rows", [False, True])
def test_plan(cuda_device, B, page, most_len, most_new, rows):
    rng = random.Random(B * 7 + page)
    lens, new, table, free = plan_case(rng, B, page, -(-(most_len + most_new) // page) + 2, most_len, most_new)
    total = sum(lens) + sum(new)
    check_plan(lens, new, table, free, len(free), page, sum(new) + rng.choice([0, 1, 5, 300]), (total + rng.choice([0, 1, 2, 3, 1030]) or 1) if rows else 0, strided=B % 2 == 1)


@pytest.mark.parametrize("B", [2390, 2448, 2457, 2458])
def test_plan_batches_around_the_default_shared_memory(cuda_device, B):
    lens, new, table, free = plan_case(random.Random(B), B, 16, 4, 30, 3)
    check_plan(lens, new, table, free, len(free), 16, sum(new), sum(lens) + sum(new))


def test_plan_long_prompts_fill_many_pages(cuda_device):
    rng = random.Random(2)
    lens, new = [5, 0, 1000], [20000, 1, 9000]
    free = list(range(5000))
    rng.shuffle(free)
    table = [[-1] * 2100 for _ in range(3)]
    for b, n in enumerate(lens):
        for i in range(-(-n // 16)):
            table[b][i] = free.pop()
    check_plan(lens, new, table, free, len(free), 16, 29001, 31000)


def test_plan_takes_a_part_of_the_free_list(cuda_device):
    check_plan([16, 3], [1, 20], [[4, -1, -1], [5, -1, -1]], [9, 8, 7, 6, 0, 1], 3, 16, 21, 0)       # free_count below the list's length
    check_plan([16, 3], [1, 20], [[4, -1, -1], [5, -1, -1]], [9, 8, 7], 90, 16, 21, 0)               # and beyond it


@pytest.mark.parametrize("change,bits", [
    (dict(free=[9]), 1), (dict(count=0), 1), (dict(count=-3), 1), (dict(table=[[4], [5]]), 2), (dict(max_tokens=20), 4), (dict(max_rows=39), 8), (dict(lens=[-1, 3]), 16),
    (dict(new=[1, -2]), 16), (dict(lens=[2147483647, 3]), 16), (dict(free=[9], max_tokens=2, max_rows=2), 13), (dict(new=[2147483000, 20]), 7)])
def test_plan_that_does_not_fit_changes_nothing(cuda_device, change, bits):
    a = dict(lens=[16, 3], new=[1, 20], table=[[4, -1, -1], [5, -1, -1]], free=[9, 8, 7], count=None, page=16, max_tokens=21, max_rows=0) | change
    if a["count"] is None:
        a["count"] = len(a["free"])
    if bits == 8:
        a["max_tokens"] = 21
    p = check_plan(*a.values())
    assert int(p.status) == bits and int(p.qo_indptr.abs().sum()) == 0 and (p.slot_map == -1).all()


def test_plan_unallocated_entry_gives_no_row(cuda_device):
    p = check_plan([20], [2], [[3, -1, -1]], [0], 1, 16, 2, 25)
    assert p.slot_map.tolist() == [-1, -1] and p.kv_indices.tolist() == list(range(48, 64)) + [-1] * 9


def test_plan_page_beyond_32_bits_of_rows(cuda_device):
    import clusterfusionplus_b200 as cf
    p = cf.paged_kv_plan(ints([20]), ints([2]), ints([[3, 1 << 28]]), ints([0]), ints([1]), 16, 2, 0)
    assert p.slot_map.tolist() == [-1, -1] and int(p.status) == 0


def test_release_returns_pages_in_order(cuda_device):
    import clusterfusionplus_b200 as cf
    table, free = ints([[4, 6, -1], [5, -1, -1], [2, 8, 1]]), ints([9, 0, 0, 0, 0, 0, 0, 0])
    left, status = cf.paged_kv_release(ints([1, 0, 7]), ints([17, 3, 33]), table, free, ints([1]), 16)
    assert int(status) == 0 and int(left) == 6 and free.tolist()[:6] == [9, 4, 6, 2, 8, 1] and table.tolist() == [[-1] * 3, [5, -1, -1], [-1] * 3]


@pytest.mark.parametrize("B", [1, 300, 4096])
def test_plan_and_release_keep_every_page_once(cuda_device, B):
    import clusterfusionplus_b200 as cf
    rng = random.Random(B)
    width, page = 6, 16
    pool = B * width + 3
    table, free = torch.full((B, width), -1, dtype=torch.int32, device=DEV), torch.randperm(pool, device=DEV).int()
    count, lens = ints([pool]), ints([0] * B)
    for _ in range(6):
        new = ints([rng.choice([0, 1, 15]) for _ in range(B)])
        p = cf.paged_kv_plan(lens, new, table, free, count, page, 15 * B)
        assert int(p.status) == 0
        done = ints([int(rng.random() < 0.3) for _ in range(B)])
        count, status = cf.paged_kv_release(done, p.kv_lens, table, free, p.free_count, page)
        assert int(status) == 0
        lens = torch.where(done != 0, torch.zeros_like(lens), p.kv_lens)
        used = table[table >= 0].tolist()
        assert sorted(used + free[:int(count)].tolist()) == list(range(pool))
        assert ((table >= 0).sum(1) == (lens + page - 1) // page).all()


@pytest.mark.parametrize("kw,bits", [(dict(free=[9, 0]), 1), (dict(count=-1), 1), (dict(lens=[17, 3, 49]), 2), (dict(lens=[-1, 3, 33]), 16), (dict(lens=[33, 3, 33]), 32)])
def test_release_that_cannot_be_changes_nothing(cuda_device, kw, bits):
    import clusterfusionplus_b200 as cf
    a = dict(lens=[17, 3, 33], free=[9] + [0] * 9, count=1) | kw
    table, free = ints([[4, 6, -1], [5, -1, -1], [2, 8, 1]]), ints(a["free"])
    left, status = cf.paged_kv_release(ints([1, 0, 1]), ints(a["lens"]), table, free, ints([a["count"]]), 16)
    assert int(status) == bits and int(left) == a["count"] and free.tolist() == a["free"] and table.tolist() == [[4, 6, -1], [5, -1, -1], [2, 8, 1]]


# -------------------------------------------------------------------------------------------------------- append, read
def rows_of(T, H, D, dtype, seed, spread=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(T, H, D, device=DEV, generator=g) * spread).to(dtype)


@pytest.mark.parametrize("T,H,D,page,dtype", [(1, 1, 16, 16, torch.float16), (3, 2, 32, 16, torch.bfloat16), (20, 3, 64, 32, torch.float16), (17, 5, 80, 48, torch.bfloat16),
                                              (40, 2, 96, 64, torch.float16), (33, 2, 128, 16, torch.bfloat16), (9, 1, 72, 128, torch.float16), (6, 2, 120, 16, torch.float16)])
def test_append_bytes(cuda_device, T, H, D, page, dtype):
    """The whole cache, byte for byte: the written rows and every other byte."""
    import clusterfusionplus_b200 as cf
    fused = rows_of(T, 3 * H, D, dtype, T * D)
    key, value = fused[:, H:2 * H], fused[:, 2 * H:]                       # rows 3 H D apart, cut out of a projection
    pages = -(-T // page) + 3
    cache = torch.randint(0, 256, (pages, H, page, 40 * S.groups(D)), dtype=torch.uint8, device=DEV)
    want = cache.cpu().numpy().copy()
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(T))[:T].tolist()
    if T > 4:
        slots[2] = -1                                                       # a padded row
    for t, s in enumerate(slots):
        if s >= 0:
            S.store(want, s, key[t].float().cpu().numpy(), value[t].float().cpu().numpy())
    cf.kv4_append(key, value, ints(slots), cache)
    assert np.array_equal(cache.cpu().numpy(), want)
    k, v = S.unpack(want, D)
    for out_dtype in (torch.float16, torch.bfloat16):
        u = torch.finfo(out_dtype).eps / 2 + 2.0 ** -24
        for got, ref in zip(cf.kv4_read(cache, ints(slots), D, out_dtype), (k, v)):
            assert got.dtype == out_dtype and got.shape == (T, H, D)
            ref = torch.stack([ref[s // page, :, s % page] if s >= 0 else torch.zeros(H, D, dtype=torch.float64) for s in slots])
            assert ((got.double().cpu() - ref).abs() <= u * ref.abs() + 2.0 ** -25).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_append_hard_values(cuda_device, dtype):
    """Constant groups, zeros, the type's largest, subnormal numbers, NaN and infinities."""
    import clusterfusionplus_b200 as cf
    D = 96
    x = rows_of(9, 1, D, dtype, 5)
    x[0] = 0
    x[1] = 1.375
    x[2, :, :32] = torch.finfo(dtype).max
    x[2, :, 32:64:2] = -torch.finfo(dtype).max
    x[3] *= 2.0 ** -22
    x[4, 0, 7] = math.nan
    x[5, 0, 40] = math.inf
    x[6, 0, 95] = -math.inf
    x[7, 0, :] = -0.0
    x[8, 0, 33] = 60000.0
    cache = cf.kv4_cache(1, 1, 16, D)
    want = cache.cpu().numpy().copy()
    for t in range(9):
        S.store(want, t, x[t].float().cpu().numpy(), x[t].float().cpu().numpy())
    cf.kv4_append(x, x, ints(list(range(9))), cache)
    k, v = cf.kv4_read(cache, ints(list(range(9))), D, torch.float16)
    rk, rv = S.unpack(want, D)
    for got, ref in ((k, rk), (v, rv)):
        got, ref = got[:, 0].double().cpu(), ref[0, 0, :9]
        assert torch.equal(got.isnan(), ref.isnan()) and got.isnan().sum() == 3 * 32
        fine = ~ref.isnan()
        assert ((got - ref).abs()[fine] <= (2.0 ** -11 + 2.0 ** -24) * ref.abs()[fine] + 2.0 ** -25).all()


def test_append_and_read_report_rows_beyond_the_cache(cuda_device):
    import clusterfusionplus_b200 as cf
    x = rows_of(3, 2, 64, torch.float16, 1)
    cache = cf.kv4_cache(2, 2, 16, 64)
    cf.kv4_append(x, x, ints([32, 5, 2147483647]), cache)
    with pytest.raises(RuntimeError, match="status 8"):
        cf.device_status()
    assert cf.device_status() == 0
    k, _ = cf.kv4_read(cache, ints([5, -1]), 64)
    assert k[0].abs().sum() > 0 and k[1].abs().sum() == 0 and (cache.view(32, -1) != 0).any()
    cf.kv4_read(cache, ints([40]), 64)
    with pytest.raises(RuntimeError, match="status 8"):
        cf.device_status()


def test_append_beyond_four_gigabytes(cuda_device):
    """Rows whose byte offsets pass 32 bits."""
    import clusterfusionplus_b200 as cf
    H, D, page = 8, 128, 64
    pages = 60000                                                            # 4.9 GB
    cache = torch.empty(pages, H, page, 160, dtype=torch.uint8, device=DEV)
    x = rows_of(3, H, D, torch.float16, 9)
    slots = ints([pages * page - 1, 3500000, 2])
    cf.kv4_append(x, x, slots, cache)
    k, v = cf.kv4_read(cache, slots, D)
    assert (k - x).abs().max() < 0.5 and torch.equal(k, v)
    table = ints([[(pages * page - 1) // page]])
    tail = rows_of(page, H, D, torch.float16, 10)
    cf.kv4_append(tail, tail, ints(list(range((pages - 1) * page, pages * page))), cache)
    q = rows_of(1, H, D, torch.float16, 11)
    got = cf.kv4_attention(q, cache, table, ints([page]))
    K, V = S.unpack(cache[-1:], D)
    close(got, S.attention(q, K, V, [[0]], [page], [0, 1], D ** -0.5), q, K, V, D ** -0.5)


# ----------------------------------------------------------------------------------------------------------- attention
def close(got, ref, query, keys, values, scale):
    u = torch.finfo(got.dtype).eps / 2
    per = query.shape[1] // keys.shape[1]
    most = keys.abs().amax((0, 2)).repeat_interleave(per, 0)                                     # [heads, D]
    e = 2.0 ** -11 * scale * (query.double().cpu().abs() * most).sum(-1, keepdim=True)
    V = values.abs().amax().item()
    bound = (2 * e + 2.0 ** -10 + 2.0 ** -16 + 2.0 ** -22) * V + u * ref.abs() + 2.0 ** -25
    d = (got.double().cpu() - ref).abs()
    assert (d <= bound).all(), (d / bound).max().item()
    if ref.numel() >= 32 and ref.norm() > 0:
        rel = ((got.double().cpu() - ref).norm() / ref.norm()).item()
        assert rel <= (1e-3 if got.dtype == torch.float16 else 2.5e-3), rel


def attention_case(lens, counts, heads, kv_heads, D, page, dtype, seed, extra_cols=1):
    g = torch.Generator(device=DEV).manual_seed(seed)
    need = [-(-max(n, 0) // page) for n in lens]
    pages = sum(need) + 3
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table, at = [], 0
    for n in need:
        table.append(perm[at:at + n] + [-1] * (max(need) - n + extra_cols))
        at += n
    cache = torch.randint(0, 256, (pages, kv_heads, page, 40 * S.groups(D)), dtype=torch.uint8, device=DEV, generator=g)
    G = S.groups(D)
    par = cache.view(pages, kv_heads, page // 16, 640 * G)[..., 512 * G:]
    n = (pages, kv_heads, page // 16, 16, 2, 1, G)
    scale, low = torch.rand(n, device=DEV, generator=g) * 0.2 + 0.15, -torch.rand(n, device=DEV, generator=g) - 1.5
    par.copy_(torch.cat([scale, low], -2).half().reshape(pages, kv_heads, page // 16, 64 * G).view(torch.uint8))
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    qkv = torch.randn(starts[-1], heads + 2 * kv_heads, D, device=DEV, generator=g).to(dtype)
    return qkv[:, :heads], cache, table, starts


@pytest.fixture(params=["by_size", "line", "prompt"])
def schedule(request, monkeypatch):
    """All three ways of doing the work: the one that the sizes choose (little work: clusters), the line of tiles with a workspace, and 128 rows at a
    time on the tensor cores, which a large hint asks for."""
    import clusterfusionplus_b200 as cf
    from clusterfusionplus_b200 import serving
    if request.param == "line":
        monkeypatch.setattr(serving, "_workspace", 64 << 20)
    if request.param == "prompt":
        plain = cf.kv4_attention
        monkeypatch.setattr(cf, "kv4_attention", lambda *a, **k: plain(*a, **(k | {"max_q_len": 4096})))


def check_attention(lens, counts, heads, kv_heads, D, page, dtype, seed=1, scale=None, max_q=None):
    import clusterfusionplus_b200 as cf
    q, cache, table, starts = attention_case(lens, counts, heads, kv_heads, D, page, dtype, seed)
    K, V = S.unpack(cache, D)
    ref = S.attention(q, K, V, table, lens, starts, D ** -0.5 if scale is None else scale)
    got = cf.kv4_attention(q, cache, ints(table), ints(lens), ints(starts), max_q_len=max(counts) if max_q is None else max_q, scale=scale)
    close(got, ref, q, K, V, D ** -0.5 if scale is None else abs(scale))
    return got


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens", [[1], [15, 16, 17], [0, 1, 300], [257, 64, 1000, 31]])
@pytest.mark.parametrize("heads,kv_heads,D,page", [(4, 4, 128, 16), (8, 2, 64, 32), (8, 1, 128, 64), (5, 1, 80, 16), (3, 3, 96, 128), (16, 1, 16, 48), (6, 3, 120, 16), (24, 1, 128, 16), (40, 1, 64, 16)])
def test_attention_of_single_tokens(cuda_device, schedule, dtype, lens, heads, kv_heads, D, page):
    check_attention(lens, [1] * len(lens), heads, kv_heads, D, page, dtype, seed=sum(lens) + heads)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lens,counts", [([5], [5]), ([40, 3, 0, 129], [2, 3, 0, 7]), ([130, 200], [130, 1]), ([64, 500], [33, 17]), ([3, 20], [6, 1]), ([300], [200]), ([0, 2], [4, 0])])
@pytest.mark.parametrize("heads,kv_heads,D,page", [(4, 4, 128, 16), (8, 2, 64, 32), (5, 1, 80, 16), (8, 1, 128, 64), (2, 2, 96, 16), (40, 2, 128, 16)])
def test_attention_of_several_queries_a_request(cuda_device, schedule, dtype, lens, counts, heads, kv_heads, D, page):
    """Drafted tokens, whole prompts, chunks behind a history; more queries than cached tokens leave rows that see nothing."""
    got = check_attention(lens, counts, heads, kv_heads, D, page, dtype, seed=sum(lens) + sum(counts))
    row = 0
    for n, c in zip(lens, counts):
        for i in range(c):
            if n - c + i < 0:
                assert (got[row + i] == 0).all()
        row += c


@pytest.mark.parametrize("max_q", [1, 3, 1000])
@pytest.mark.parametrize("lens,counts", [([40, 300], [2, 150]), ([600, 7], [1, 1])])
def test_attention_does_not_depend_on_the_hint(cuda_device, schedule, max_q, lens, counts):
    check_attention(lens, counts, 8, 2, 128, 16, torch.float16, max_q=max_q)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.25, 3.0])
def test_attention_scale(cuda_device, schedule, scale):
    check_attention([70, 9], [3, 1], 4, 2, 64, 16, torch.float16, scale=scale)


@pytest.mark.parametrize("counts", [[1], [9], [140]])
def test_attention_long_cache(cuda_device, schedule, counts):
    check_attention([20000], counts, 2, 1, 64, 64, torch.float16)


def test_attention_many_requests(cuda_device, schedule):
    rng = random.Random(4)
    lens = [rng.randint(0, 90) for _ in range(700)]
    check_attention(lens, [min(1, n) for n in lens], 2, 1, 64, 16, torch.float16)


def test_attention_of_uneven_requests(cuda_device, schedule):
    """Pieces of the line that begin and end everywhere: one long request among many short ones, ends on and off the tiles' borders."""
    check_attention([1, 5000, 16, 0, 17, 300, 1600, 1], [1, 1, 1, 1, 1, 1, 1, 0], 8, 4, 128, 16, torch.float16, seed=2)
    check_attention([64] * 40, [1] * 40, 4, 4, 64, 32, torch.bfloat16, seed=3)
    check_attention([7000, 3, 900], [2, 3, 1], 16, 2, 96, 48, torch.float16, seed=4)


def test_attention_of_long_prompts(cuda_device):
    """The tensor cores' way chosen by the sizes: several tiles of rows, ends off the tiles' borders, a length that the last tile does not fill."""
    check_attention([700, 333], [700, 200], 8, 2, 128, 16, torch.bfloat16, seed=7)
    check_attention([1100], [513], 4, 4, 80, 48, torch.float16, seed=8)
    check_attention([260, 5, 0, 129], [129, 5, 0, 129], 16, 2, 64, 32, torch.float16, seed=9)


def test_attention_chooses_the_line_by_itself(cuda_device):
    from clusterfusionplus_b200._lib import lib
    assert lib.cf_kv4_attention_workspace(2, 8, 8, 128, 16384, 1) > 0 and lib.cf_kv4_attention_workspace(1, 8, 8, 128, 1024, 1) == 0
    check_attention([16000, 9000], [1, 1], 8, 8, 128, 64, torch.float16, seed=6)


@pytest.mark.parametrize("counts", [[1, 1, 1], [5, 70, 1]])
def test_attention_leaves_other_rows(cuda_device, schedule, counts):
    """Rows before the first request's and behind the last one's stay as they were, and padded requests own none."""
    import clusterfusionplus_b200 as cf
    q, cache, table, starts = attention_case([30, 90, 2], counts, 4, 2, 64, 16, torch.float16, 3)
    n = starts[-1]
    pad = torch.cat([q.new_zeros(2, 4, 64), q, q.new_zeros(5, 4, 64)])
    out = torch.full((n + 7, 4, 64), 7.0, device=DEV, dtype=torch.float16)
    back = cf.kv4_attention(pad, cache, ints(table + [[-1] * len(table[0])] * 2), ints([30, 90, 2, 0, 0]), ints([s + 2 for s in starts] + [n + 2] * 2), max_q_len=max(counts), out=out)
    assert back is out and (out[:2] == 7).all() and (out[n + 2:] == 7).all()
    K, V = S.unpack(cache, 64)
    close(out[2:n + 2], S.attention(q, K, V, table, [30, 90, 2], starts, 0.125), q, K, V, 0.125)


@pytest.mark.parametrize("counts", [[1, 1], [20, 90]])
def test_attention_skips_and_reports_bad_pages(cuda_device, schedule, counts):
    import clusterfusionplus_b200 as cf
    q, cache, table, starts = attention_case([100, 130], counts, 4, 2, 128, 16, torch.float16, 8)
    table[0][2], table[1][1], table[1][5] = -5, cache.shape[0], 2147483647
    K, V = S.unpack(cache, 128)
    got = cf.kv4_attention(q, cache, ints(table), ints([100, 130]), ints(starts), max_q_len=max(counts))
    with pytest.raises(RuntimeError, match="status 8"):
        cf.device_status()
    close(got, S.attention(q, K, V, table, [100, 130], starts, 128 ** -0.5), q, K, V, 128 ** -0.5)
    # a length beyond the table: what the table names is there
    got = cf.kv4_attention(q[:1], cache, ints([table[0][:2]]), ints([5000]))
    close(got, S.attention(q[:1], K, V, [table[0][:2]], [32], [0, 1], 128 ** -0.5), q[:1], K, V, 128 ** -0.5)


@pytest.mark.parametrize("count", [1, 7, 80])
def test_attention_ignores_what_lies_behind_the_last_token(cuda_device, schedule, count):
    """Stale NaN and infinities in the rows behind a request's end and in its page's other rows."""
    import clusterfusionplus_b200 as cf
    q, cache, table, starts = attention_case([83], [count], 4, 2, 128, 32, torch.float16, 21)
    K, V = S.unpack(cache, 128)
    K, V = K.clone(), V.clone()
    ref = S.attention(q, K, V, table, [83], starts, 128 ** -0.5)
    flat = cache.view(-1, 2, 2, 2560)
    last, junk = table[0][2], torch.tensor([math.nan, math.inf, -math.inf, 65504.0], dtype=torch.float16, device=DEV)
    par = flat[last, :, 1, 2048:].view(torch.float16).view(2, 16, 16)                            # token 80 .. 95 of the request
    par[:, 3:] = junk.repeat(4)
    got = cf.kv4_attention(q, cache, ints(table), ints([83]), ints(starts), max_q_len=count)
    close(got, ref, q, K, V, 128 ** -0.5)


@pytest.mark.parametrize("count", [1, 40])
def test_attention_passes_on_nan_that_it_sees(cuda_device, schedule, count):
    import clusterfusionplus_b200 as cf
    q, cache, table, starts = attention_case([60, 60], [count, count], 2, 2, 64, 16, torch.float16, 22)
    x = rows_of(1, 2, 64, torch.float16, 3)
    x[0, 1, 5] = math.nan
    cf.kv4_append(x, rows_of(1, 2, 64, torch.float16, 4), ints([table[0][0] * 16]), cache)       # token 0 of request 0, head 1
    got = cf.kv4_attention(q, cache, ints(table), ints([60, 60]), ints(starts), max_q_len=count)
    assert got[:count, 1].isnan().all() and not got[:count, 0].isnan().any() and not got[count:].isnan().any()


@pytest.mark.parametrize("size", [2.0 ** -14, 2.0 ** -6, 200.0, 5000.0])
@pytest.mark.parametrize("count", [1, 30])
def test_attention_of_small_and_large_values(cuda_device, schedule, size, count):
    """Values from fp16's smallest normal number to thousands; keys of unit size."""
    import clusterfusionplus_b200 as cf
    D, T = 128, 150
    q, key = rows_of(count, 4, D, torch.float16, 1), rows_of(T, 2, D, torch.float16, 2)
    value = rows_of(T, 2, D, torch.float16, 3, spread=size)
    cache = cf.kv4_cache(10, 2, 16, D)
    cf.kv4_append(key, value, ints(list(range(T))), cache)
    K, V = S.unpack(cache, D)
    table = [list(range(10))]
    got = cf.kv4_attention(q, cache, ints(table), ints([T]), ints([0, count]), max_q_len=count)
    ref = S.attention(q, K, V, table, [T], [0, count], D ** -0.5)
    assert ((got.double().cpu() - ref).norm() / ref.norm()).item() <= (1e-3 if size > 2.0 ** -10 else 5e-3)   # 2^-14: results are subnormal fp16 numbers, steps of 2^-24


@pytest.mark.parametrize("size", [1e-3, 40.0, 3000.0])
def test_attention_of_small_and_large_queries(cuda_device, schedule, size):
    """Large queries make one-hot probabilities; bf16 queries reach beyond fp16."""
    import clusterfusionplus_b200 as cf
    D = 64
    q, cache, table, starts = attention_case([200], [3], 4, 2, D, 16, torch.bfloat16, 31)
    K, V = S.unpack(cache, D)
    for f in (size, size * 2.0 ** 60):
        x = (q.float() * f).to(torch.bfloat16)
        scale = D ** -0.5 / size * (1 if f == size else 2.0 ** -60)
        got = cf.kv4_attention(x, cache, ints(table), ints([200]), ints(starts), max_q_len=3, scale=scale)
        close(got, S.attention(x, K, V, table, [200], starts, scale), x, K, V, scale)


def test_attention_refuses(cuda_device):
    import clusterfusionplus_b200 as cf
    q, cache, table, starts = attention_case([30], [1], 4, 2, 64, 16, torch.float16, 3)
    t, n = ints(table), ints([30])
    for call, match in [
            (lambda: cf.kv4_attention(q.float(), cache, t, n), "dtype"), (lambda: cf.kv4_attention(q[..., :63], cache, t, n), "head_dim"),
            (lambda: cf.kv4_attention(q, cache[:, :1], t, n), "contiguous"), (lambda: cf.kv4_attention(q[:, :3], cache, t, n), "query heads"),
            (lambda: cf.kv4_attention(q, cache, t.long(), n), "int32"), (lambda: cf.kv4_attention(q, cache, t, n.long()), "int32"), (lambda: cf.kv4_attention(q, cache, t, n, ints([0])), "entries"),
            (lambda: cf.kv4_attention(q.cpu(), cache, t, n), "CUDA tensor"), (lambda: cf.kv4_attention(q.transpose(0, 1), cache, t, n), "query heads"),
            (lambda: cf.kv4_attention(q, cache, t, n, max_q_len=0), "max_q_len"), (lambda: cf.kv4_attention(q, cache, t, n, out=q.new_empty(1, 4, 32)), "out"),
            (lambda: cf.kv4_attention(q[:0], cache, t, n), "query rows"), (lambda: cf.kv4_append(q, q[:, :2], ints([0]), cache), "value"), (lambda: cf.kv4_append(q[:, :2], q[:, :2], ints([0, 1]), cache), "entries"),
            (lambda: cf.kv4_read(cache, ints([0]), 96), "cache"), (lambda: cf.kv4_read(cache, ints([0]), 64, torch.float32), "dtype"),
            (lambda: cf.paged_kv_plan(n, ints([1, 2]), t, n, n, 16, 3), "entries"), (lambda: cf.paged_kv_plan(n, n, t.t(), n, n, 16, 3), "block_table"), (lambda: cf.paged_kv_plan(n, n, t, n, n, 16, -1), "negative")]:
        with pytest.raises(RuntimeError, match=match):
            call()


# ---------------------------------------------------------------------------------------------------- log probabilities
def check_logprobs(x, tokens, k, token_dtype=torch.int64):
    import clusterfusionplus_b200 as cf
    got = cf.token_logprobs(x, torch.tensor(tokens, dtype=token_dtype, device=DEV), k)
    lp, h, tl, ti = S.logprobs(x, tokens, k)
    assert got.top_tokens.tolist() == ti.tolist()
    n = x.shape[1]
    rel = 2 * (n / 512 + 28) * 2.0 ** -24
    for a, b in ((got.logprobs, lp), (got.entropy, h), (got.top_logprobs, tl)):
        a = a.double().cpu()
        assert a.shape == b.shape and torch.equal(a.isnan(), b.isnan())
        fine = b.isfinite()
        assert torch.equal(a[~fine & ~b.isnan()], b[~fine & ~b.isnan()])
        assert ((a - b).abs()[fine] <= rel * b.abs()[fine].clamp(min=12.0)).all(), ((a - b).abs()[fine] / (rel * b.abs()[fine].clamp(min=12.0))).max()
    return got


def logits(rows, vocab, dtype, seed, pad=0, spread=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(rows, vocab + pad, device=DEV, generator=g) * spread).to(dtype)[:, :vocab]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,pad,k", [(1, 1, 0, 1), (3, 2, 0, 2), (2, 7, 1, 7), (5, 33, 0, 32), (4, 511, 1, 20), (1, 4097, 3, 5), (1, 50304, 0, 32), (7, 8193, 1, 1), (160, 300, 5, 4), (3, 32000, 0, 0), (37, 20001, 2, 20)])
def test_logprobs(cuda_device, dtype, rows, vocab, pad, k):
    rng = random.Random(vocab)
    check_logprobs(logits(rows, vocab, dtype, rows + vocab, pad), [rng.randrange(vocab) for _ in range(rows)], k, rng.choice([torch.int32, torch.int64]))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [600, 20000])
def test_logprobs_ties_go_to_the_lower_token(cuda_device, dtype, vocab):
    x = logits(6, vocab, dtype, 3)
    x[0] = 0                                                   # all equal
    x[1] = torch.round(x[1].float()).to(dtype)                 # a few values only
    x[2, ::2], x[2, 1::2] = 0.0, -0.0                          # -0 equals +0
    x[3] = torch.arange(vocab, device=DEV).to(dtype)           # ascending (the 16-bit types with ties)
    x[4] = -torch.arange(vocab, device=DEV).to(dtype)
    x[5, 512 * 4::512 * 8] = 30.0                              # all of the top in few threads' shares
    check_logprobs(x, [0, 5, vocab - 1, vocab - 1, 0, 9], 32)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_logprobs_orders_that_crowd_one_share(cuda_device, dtype):
    """Ever greater values at the places that a few threads read."""
    vocab, E = 200000, 4 if dtype == torch.float32 else 8
    x = logits(1, vocab, dtype, 3, spread=0.5)
    for t in range(40):
        at = torch.arange(t * E, vocab, 512 * E, device=DEV)
        for e in range(E):
            x[0, at + e] = (20 + torch.arange(at.numel(), device=DEV) * 0.25).to(dtype)
    check_logprobs(x.repeat(200, 1)[:, :150000], [0] * 200, 32)
    check_logprobs(x, [7], 32)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [50, 9000])
def test_logprobs_masks_and_broken_rows(cuda_device, dtype, vocab):
    """-inf and the type's lowest value as masks, rows that are all one of them, infinities, NaN, tokens outside the vocabulary."""
    x = logits(12, vocab, dtype, 9)
    low = torch.finfo(dtype).min
    x[0, 10:] = -math.inf
    x[1, 10:] = low
    x[2] = -math.inf
    x[3] = low
    x[4, :], x[4, 17] = -math.inf, low                         # one number, the lowest
    x[5, 20] = math.inf
    x[6, 20], x[6, 3] = math.nan, math.nan
    x[7, 20], x[7, 21] = math.inf, math.nan
    x[8, 3] = torch.finfo(dtype).max
    x[9, ::3] = -math.inf
    x[10] = torch.finfo(dtype).max
    got = check_logprobs(x, [3, 12, 0, 1, 17, 20, 1, 2, 3, 0, 4, vocab], 5)
    assert got.logprobs[11] == -math.inf
    assert check_logprobs(x[9:10], [-1], 0).logprobs[0] == -math.inf


def test_logprobs_large_logits_keep_their_precision(cuda_device):
    x = logits(4, 5000, torch.float32, 2) + torch.tensor([[1e4], [-1e5], [0.0], [3e6]], device=DEV)
    check_logprobs(x, [1, 2, 3, 4], 8)


@pytest.mark.parametrize("dtype,vocab", [(torch.float16, v) for v in (2040, 2047, 2048, 2049, 2063)] + [(torch.float32, v) for v in (1020, 1024, 1027)])
@pytest.mark.parametrize("k", [1, 10, 11])
def test_logprobs_where_every_thread_just_has_elements(cuda_device, dtype, vocab, k):
    """256 threads of one 16-byte vector each, give or take one: the bound of the top k comes from more or fewer groups of them."""
    check_logprobs(logits(3, vocab, dtype, vocab + k, pad=3), [0, vocab - 1, vocab // 2], k)


def test_logprobs_of_one_vector_and_of_none(cuda_device):
    import clusterfusionplus_b200 as cf
    x = logits(1, 1000, torch.float32, 2)
    a, b = cf.token_logprobs(x[0], torch.tensor([4], device=DEV), 3), cf.token_logprobs(x, torch.tensor([4], device=DEV), 3)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    none = cf.token_logprobs(x[:0], torch.zeros(0, dtype=torch.int64, device=DEV), 3)
    assert none.logprobs.shape == (0,) and none.top_tokens.shape == (0, 3)
    same = cf.token_logprobs(x.expand(3, -1), torch.tensor([4, 5, 4], device=DEV), 3)              # rows 0 elements apart
    assert same.logprobs[0] == same.logprobs[2] == a.logprobs[0]


def test_logprobs_refuses(cuda_device):
    import clusterfusionplus_b200 as cf
    x, t = logits(2, 100, torch.float32, 1), torch.tensor([1, 2], device=DEV)
    for call, match in [(lambda: cf.token_logprobs(x.double(), t), "logits"), (lambda: cf.token_logprobs(x.t(), t), "last axis"), (lambda: cf.token_logprobs(x, t[:1]), "tokens"),
                        (lambda: cf.token_logprobs(x, t.float()), "tokens"), (lambda: cf.token_logprobs(x, t, 33), "top_k"), (lambda: cf.token_logprobs(x[:, :4], t, 5), "top_k"),
                        (lambda: cf.token_logprobs(x.cpu(), t), "CUDA tensor"), (lambda: cf.token_logprobs(x, t, -1), "top_k")]:
        with pytest.raises(RuntimeError, match=match):
            call()


# ------------------------------------------------------------------------------------------------------------ together
def serving_state(B, H, Hkv, D, page, prompt, seed=1):
    import clusterfusionplus_b200 as cf
    pool = 40 * B
    g = torch.Generator(device=DEV).manual_seed(seed)
    return dict(table=torch.full((B, 24), -1, dtype=torch.int32, device=DEV), free=torch.randperm(pool, device=DEV, generator=g).int(), count=ints([pool]),
                lens=ints([0] * B), cache=cf.kv4_cache(pool, Hkv, page, D), g=g)


@pytest.mark.parametrize("dtype,H,Hkv,D", [(torch.float16, 4, 4, 128), (torch.bfloat16, 8, 2, 80)])
def test_serving_steps(cuda_device, schedule, dtype, H, Hkv, D):
    """Prompts, then single tokens, then a request that ends and one that takes its place, all through plan, append and attention, with log
    probabilities of what a head makes of the result; compared with dense attention over what was written."""
    import clusterfusionplus_b200 as cf
    B, page, vocab = 3, 16, 200
    s = serving_state(B, H, Hkv, D, page, 50)
    head = torch.randn(H * D, vocab, device=DEV, generator=s["g"])
    steps = [([50, 17, 1], [0, 0, 0]), ([1, 1, 1], [0, 0, 0]), ([1, 0, 5], [0, 1, 0]), ([1, 33, 1], [0, 0, 0])]
    kept = [[] for _ in range(B)]
    free_now = s["free"].numel()
    for new, done in steps:
        p = cf.paged_kv_plan(s["lens"], ints(new), s["table"], s["free"], s["count"], page, 80)
        assert int(p.status) == 0
        n = sum(new)
        qkv = torch.randn(80, H + 2 * Hkv, D, device=DEV, generator=s["g"]).to(dtype)
        key, value = qkv[:, H:H + Hkv], qkv[:, H + Hkv:]
        cf.kv4_append(key, value, p.slot_map, s["cache"])                                       # the padded rows are skipped
        out = cf.kv4_attention(qkv[:, :H], s["cache"], s["table"], p.kv_lens, p.qo_indptr, max_q_len=max(new))
        row = 0
        for b, c in enumerate(new):
            for i in range(c):
                kept[b].append((key[row], value[row]))
                row += 1
        assert p.kv_lens.tolist() == [len(x) for x in kept]
        # dense: what was written, quantised by the oracle
        row = 0
        for b, c in enumerate(new):
            if c:
                dense = np.zeros((1, Hkv, -(-len(kept[b]) // 16) * 16, 40 * S.groups(D)), np.uint8)
                for i, (k, v) in enumerate(kept[b]):
                    S.store(dense, i, k.float().cpu().numpy(), v.float().cpu().numpy())
                K, V = S.unpack(dense, D)
                ref = S.attention(qkv[row:row + c, :H], K, V, [[0]], [len(kept[b])], [0, c], D ** -0.5)
                close(out[row:row + c], ref, qkv[row:row + c, :H], K, V, D ** -0.5)
            row += c
        lg = (out[:n].flatten(1).float() @ head).contiguous()
        check_logprobs(lg, [i % vocab for i in range(n)], 4)
        s["count"], status = cf.paged_kv_release(ints(done), p.kv_lens, s["table"], s["free"], p.free_count, page)
        assert int(status) == 0
        s["lens"] = torch.where(ints(done) != 0, torch.zeros_like(p.kv_lens), p.kv_lens)
        kept = [[] if d else x for d, x in zip(done, kept)]
        assert int(s["count"]) == free_now - sum(-(-len(x) // page) for x in kept)


def test_serving_step_captured_and_replayed(cuda_device):
    """The whole step in one CUDA graph: lengths, tables and the free list live on the device and advance with every replay.  A second graph
    over other tensors, replayed in between on another stream, does not disturb it."""
    import clusterfusionplus_b200 as cf
    B, H, Hkv, D, page, vocab = 4, 8, 2, 64, 16, 500

    def build(seed):
        s = serving_state(B, H, Hkv, D, page, 1, seed)
        s["qkv"] = torch.randn(B, H + 2 * Hkv, D, device=DEV, generator=s["g"]).half()
        s["new"], s["head"] = ints([1] * B), torch.randn(H * D, vocab, device=DEV, generator=s["g"]).half()
        s["tokens"] = ints([3, 1, 4, 1])

        def step():
            p = cf.paged_kv_plan(s["lens"], s["new"], s["table"], s["free"], s["count"], page, B, 512)
            cf.kv4_append(s["qkv"][:, H:H + Hkv], s["qkv"][:, H + Hkv:], p.slot_map, s["cache"])
            out = cf.kv4_attention(s["qkv"][:, :H], s["cache"], s["table"], p.kv_lens, p.qo_indptr)
            s["lens"].copy_(p.kv_lens)
            s["count"].copy_(p.free_count)
            return p, out, cf.token_logprobs(out.flatten(1) @ s["head"], s["tokens"], 3)
        return s, step

    def run_eager(seed, steps):
        s, step = build(seed)
        for i in range(steps):
            s["qkv"].copy_(inputs(seed, i, s["qkv"]))
            p, out, lp = step()
        return [x.clone() for x in (p.kv_lens, p.slot_map, p.kv_indices, out, lp.logprobs, lp.entropy, lp.top_tokens, s["table"], s["cache"])]

    def inputs(seed, i, like):
        g = torch.Generator(device=DEV).manual_seed(seed * 1000 + i)
        return torch.randn(like.shape, device=DEV, generator=g).half()

    graphs = []
    for seed in (1, 2):
        s, step = build(seed)
        keep = {k: s[k].clone() for k in ("lens", "count", "table", "cache")}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            result = step()
        for k, v in keep.items():
            s[k].copy_(v)
        graphs.append((seed, s, g, result, torch.cuda.Stream()))
    torch.cuda.synchronize()
    steps = 37
    for i in range(steps):
        for seed, s, g, _, stream in graphs:
            with torch.cuda.stream(stream):
                s["qkv"].copy_(inputs(seed, i, s["qkv"]))
                g.replay()
    torch.cuda.synchronize()
    for seed, s, g, (p, out, lp), _ in graphs:
        want = run_eager(seed, steps)
        got = (p.kv_lens, p.slot_map, p.kv_indices, out, lp.logprobs, lp.entropy, lp.top_tokens, s["table"], s["cache"])
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_attention_with_ctas_that_have_nothing_to_read(cuda_device):
    """A wide block table asks for clusters of 8 CTAs; requests of 0, 1 and 17 tokens, and without queries, leave most of them nothing to do but
    send their empty results to the others."""
    import clusterfusionplus_b200 as cf
    lens, counts = [1, 0, 17, 1, 300, 2, 1, 1], [1, 1, 1, 0, 1, 1, 0, 1]
    q, cache, table, starts = attention_case(lens, counts, 4, 2, 64, 16, torch.float16, 21)
    wide = [row + [-1] * (4096 - len(row)) for row in table]
    K, V = S.unpack(cache, 64)
    ref = S.attention(q, K, V, table, lens, starts, 64 ** -0.5)
    for _ in range(20):
        close(cf.kv4_attention(q, cache, ints(wide), ints(lens), ints(starts)), ref, q, K, V, 64 ** -0.5)


def test_calls_on_two_streams_do_not_disturb_each_other(cuda_device, schedule):
    import clusterfusionplus_b200 as cf
    cases = []
    for seed, lens in ((1, [5000, 40, 700]), (2, [90, 6000, 1])):
        q, cache, table, starts = attention_case(lens, [1, 3, 1], 8, 2, 128, 16, torch.float16, seed)
        cases.append((q, cache, ints(table), ints(lens), ints(starts)))
    want = [cf.kv4_attention(*c, max_q_len=3) for c in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(50):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(cf.kv4_attention(*cases[i], max_q_len=3))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in (0, 1) for x in got[i])


def test_calls_of_two_threads(cuda_device):
    """Each on a stream of its own; one thread's refusals do not reach the other."""
    import threading

    import clusterfusionplus_b200 as cf
    want, got, errors = [], [[], []], []
    cases = [attention_case(lens, [1, 1], 8, 2, 64, 16, torch.float16, seed) for seed, lens in ((1, [700, 30]), (2, [9, 1200]))]
    args = [(q, cache, ints(table), ints(lens)) for (q, cache, table, _), lens in zip(cases, ([700, 30], [9, 1200]))]
    want = [cf.kv4_attention(*a) for a in args]
    torch.cuda.synchronize()

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(200):
                    got[i].append(cf.kv4_attention(*args[i]))
                    with pytest.raises(RuntimeError, match="page size" if i else "max_q_len"):
                        cf.paged_kv_plan(args[i][3], args[i][3], args[i][2], args[i][3], args[i][3][:1], 0, 4) if i else cf.kv4_attention(*args[i], max_q_len=0)
                torch.cuda.current_stream().synchronize()
        except BaseException as e:  # noqa: BLE001 (handed to the test's own thread)
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in (0, 1)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors, errors
    assert all(len(got[i]) == 200 and torch.equal(x, want[i]) for i in (0, 1) for x in got[i])


def test_first_calls_of_a_process_inside_a_capture(cuda_device):
    """Nothing that a first call sets up (kernel attributes, addresses) is forbidden while a stream is captured."""
    import subprocess
    import sys
    code = """
import torch
import clusterfusionplus_b200 as cf
dev = torch.device("cuda:0")
i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device=dev)
cached, new, free, count, table = i32(200, 3), i32(1, 1), torch.arange(40, dtype=torch.int32, device=dev), i32(10), torch.zeros(2, 16, dtype=torch.int32, device=dev)
table[0] = torch.arange(40, 56, device=dev)
table[1] = torch.arange(56, 72, device=dev)
cache, x = cf.kv4_cache(72, 2, 16, 64), torch.ones(2, 12, 64, dtype=torch.float16, device=dev)
many, starts, logits = torch.ones(140, 8, 64, dtype=torch.float16, device=dev), i32(0, 139, 140), torch.zeros(2, 50304, device=dev)
big, wide = cf.kv4_cache(72, 8, 1024, 64), torch.ones(2, 8, 64, dtype=torch.float16, device=dev)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    p = cf.paged_kv_plan(cached, new, table, free, count, 16, 2, 300)
    cf.kv4_append(x[:, 8:10], x[:, 10:], p.slot_map, cache)
    k, v = cf.kv4_read(cache, p.slot_map, 64)
    a = cf.kv4_attention(x[:, :8], cache, table, p.kv_lens)
    b = cf.kv4_attention(many, cache, table, p.kv_lens, starts, max_q_len=139)
    c = cf.kv4_attention(wide, big, table, p.kv_lens)
    s = cf.token_logprobs(logits, new, 3)
    left, status = cf.paged_kv_release(new, p.kv_lens, table, free, p.free_count, 16)
g.replay()  # once: its last call gives the pages back
torch.cuda.synchronize()
assert bool((k == 1).all()) and bool((v == 1).all()) and int(status) == 0, (k, v, status)
assert abs(float(s.entropy[0]) - 10.82584) < 1e-4, s.entropy
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr


def test_attention_of_shared_pages(cuda_device, schedule):
    """Requests with a common prefix name the same pages."""
    import clusterfusionplus_b200 as cf
    q, cache, table, starts = attention_case([300, 300], [1, 1], 8, 2, 64, 16, torch.float16, 12)
    shared = [table[0], table[0][:10] + table[1][10:]]
    K, V = S.unpack(cache.cpu().numpy(), 64)
    out = cf.kv4_attention(q, cache, ints(shared), ints([300, 290]), ints(starts))
    close(out, S.attention(q, K, V, shared, [300, 290], starts, 64 ** -0.5), q, K, V, 64 ** -0.5)


def test_offsets_beyond_32_bits(cuda_device):
    """Rows of queries, keys and logits that lie more than 2^31 elements apart."""
    import clusterfusionplus_b200 as cf
    apart = 1 << 30
    room = torch.empty(2 * apart + 60000, dtype=torch.float16, device=DEV)
    q, cache, table, starts = attention_case([300, 20, 77], [1, 1, 1], 8, 2, 64, 16, torch.float16, 13)
    far = room.as_strided((3, 8, 64), (apart, 64, 1))
    far.copy_(q)
    n = ints([300, 20, 77])
    assert torch.equal(cf.kv4_attention(far, cache, ints(table), n), cf.kv4_attention(q, cache, ints(table), n))
    one, two = cache.clone(), cache.clone()
    cf.kv4_append(far[:, :2], far[:, 2:4], ints([5, 6, 7]), one)
    cf.kv4_append(q[:, :2], q[:, 2:4], ints([5, 6, 7]), two)
    assert torch.equal(one, two)
    x = logits(3, 50301, torch.float16, 5)
    far = room.as_strided((3, 50301), (apart, 1))
    far.copy_(x)
    check_logprobs(far, [1, 2, 50300], 5)  # to 64-bit numbers: where a row starts within 16 bytes decides the order of its sums


def test_results_carry_no_gradient(cuda_device):
    import clusterfusionplus_b200 as cf
    x = logits(2, 100, torch.float32, 3).requires_grad_()
    assert not any(t.requires_grad for t in cf.token_logprobs(x, ints([1, 2]), 2))
    with torch.inference_mode():
        assert torch.equal(cf.token_logprobs(x, ints([1, 2]), 2).logprobs, cf.token_logprobs(x.detach(), ints([1, 2]), 2).logprobs)


def test_results_are_the_same_every_time(cuda_device):
    import clusterfusionplus_b200 as cf
    q, cache, table, starts = attention_case([3000, 100, 900], [1, 1, 1], 8, 2, 128, 16, torch.float16, 5)
    runs = [cf.kv4_attention(q, cache, ints(table), ints([3000, 100, 900]), ints(starts)) for _ in range(5)]
    x = logits(2, 50304, torch.float16, 4)
    lps = [cf.token_logprobs(x, ints([5, 6]), 20) for _ in range(5)]
    assert all(torch.equal(r, runs[0]) for r in runs) and all(torch.equal(a, b) for l in lps for a, b in zip(l, lps[0]))


def test_plan_rows_drive_the_paged_llama_block(cuda_device):
    """kv_indptr, kv_indices and positions of a plan are what llama_decoder_layer_batch_decode_sglang reads."""
    import clusterfusionplus_b200 as cf
    from oracle import llama_oracle as LO
    from oracle import pythia_oracle as O
    B, page, H = 3, 16, 4096
    lens, table, free = [40, 0, 16], [[4, 1, 0], [-1] * 3, [7, -1, -1]], list(range(8, 12))
    p = cf.paged_kv_plan(ints(lens), ints([1] * B), ints(table), ints(free), ints([4]), page, B, 60)
    pool = 12 * page
    kp, vp = O.seeded_normal((pool, H), 1, device=DEV), O.seeded_normal((pool, H), 2, device=DEV)
    x, res = O.seeded_normal((B, H), 3, device=DEV), O.seeded_normal((B, H), 4, device=DEV)
    wqkv, wo = O.seeded_normal((3 * H, H), 5, std=0.02, device=DEV), O.seeded_normal((H, H), 6, std=0.02, device=DEV)
    g1 = O.seeded_normal((H,), 7, mean=1.0, std=0.02, device=DEV)
    inv = 1.0 / (10000.0 ** (torch.arange(0, 128, 2, dtype=torch.float32) / 128))
    ang = torch.outer(torch.arange(64, dtype=torch.float32), inv)
    cs = torch.cat([ang.cos(), ang.sin()], dim=1).contiguous().to(DEV)
    k0, v0 = kp.clone(), vp.clone()
    out, res_out = torch.empty_like(x), torch.empty_like(x)
    ptr = lambda t: torch.tensor([t.data_ptr()], dtype=torch.int64, device=DEV)  # noqa: E731
    cf.llama_decoder_layer_batch_decode_sglang(out, res_out, x, res, wqkv, wo, p.kv_indptr.clone(), p.kv_indices.clone(), ptr(kp), ptr(vp), 0, g1, 1e-5, p.positions, cs)
    ro, _, rk, _, slots = LO.llama_attn_block_batch_fp32(x, res, wqkv, wo, k0, v0, p.kv_indptr, p.kv_indices, p.positions, cs, g1, 1e-5)
    assert slots.tolist() == p.slot_map.tolist()
    mx, rl = O.compare(out, ro)
    assert mx <= 2e-2 and rl <= 1e-3


def test_score_of_a_prompt(cuda_device):
    """PythiaDecoder.score: the log probabilities of a prompt's tokens against the decoder's own fp32 logits, token by token."""
    import clusterfusionplus_b200 as cf
    from oracle import pythia_oracle as O
    mini = O.Shape("mini", hidden=512, heads=4, head_dim=128, rotary=32, ffn=2048, vocab=1024, layers=2)
    layers = [O.make_layer_weights(mini, l, seed=5, device=DEV, std=0.05) for l in range(mini.layers)]
    head = O.make_head_weights(mini, seed=5, device=DEV, std=0.05)
    d = cf.CfDims()
    d.hidden, d.heads, d.head_dim, d.rotary, d.ffn, d.vocab = 512, 4, 128, 32, 2048, 1024
    caches = [(torch.zeros(64, 512, dtype=torch.float16, device=DEV), torch.zeros(64, 512, dtype=torch.float16, device=DEV)) for _ in layers]
    dec = cf.PythiaDecoder(d, layers, head, caches, 64, use_graph=False)
    rng = random.Random(1)
    tokens = [rng.randrange(1024) for _ in range(24)]
    got = dec.score(tokens, 5)
    dec.step()
    after = int(dec.token.item())
    assert got.logprobs.shape == (23,) and got.top_tokens.shape == (23, 5)
    dec.reset(0, tokens[0])
    rows = []
    for t in tokens[1:]:
        dec.step()
        rows.append(dec.logits.clone())
        one = cf.token_logprobs(dec.logits, dec.token, 3)      # the token the decoder chose is the most probable one
        assert int(one.top_tokens[0, 0]) == int(dec.token) and one.logprobs[0] == one.top_logprobs[0, 0]
        dec.token.fill_(t)
    lp, h, tl, _ = S.logprobs(torch.stack(rows), tokens[1:], 5)
    # both passes round their activations to fp16 in other places: the project's parity bar for logits-sized numbers (2e-2), twice
    assert (got.logprobs.double().cpu() - lp).abs().max() <= 4e-2 and (got.entropy.double().cpu() - h).abs().max() <= 4e-2
    assert (got.top_logprobs.double().cpu() - tl).abs().max() <= 4e-2
    dec.reset(len(tokens) - 1, tokens[-1])
    dec.step()
    assert int(dec.token.item()) == after
    assert dec.score(tokens[:1], 2).top_tokens.shape == (0, 2)
    dec.close()
