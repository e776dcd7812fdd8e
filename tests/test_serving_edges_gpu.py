"""Calls of the serving operators, and of the paged Llama block behind a step plan, that their documentation allows and that lie at the edges:
lists of a plan that did not fit, idle requests, pages that were never given, values next to a type's largest."""
import math
import random

import pytest
import torch

from oracle import llama_oracle as LO
from oracle import pythia_oracle as O
from oracle import serving_oracle as S

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
H = 4096


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.fixture(autouse=True)
def clean_status(cuda_device):
    import clusterfusionplus_b200 as cf
    yield
    torch.cuda.synchronize()
    assert cf.device_status() == 0


# ------------------------------------------------------------------------------------------- the paged Llama block's lists
@pytest.fixture(scope="module")
def llama(cuda_device):
    inv = 1.0 / (10000.0 ** (torch.arange(0, 128, 2, dtype=torch.float32) / 128))
    ang = torch.outer(torch.arange(512, dtype=torch.float32), inv)
    return dict(wqkv=O.seeded_normal((3 * H, H), 5, std=0.02, device=DEV), wo=O.seeded_normal((H, H), 6, std=0.02, device=DEV),
                g=O.seeded_normal((H,), 7, mean=1.0, std=0.02, device=DEV), cs=torch.cat([ang.cos(), ang.sin()], dim=1).contiguous().to(DEV))


class Pools:
    """Key and value rows with two more ahead of them and behind them, which nothing may touch."""

    def __init__(self, rows):
        self.room = [O.seeded_normal((rows + 4, H), seed, device=DEV) for seed in (1, 2)]
        self.before = [r.clone() for r in self.room]
        self.pools = [r[2:-2] for r in self.room]
        self.start = [p.clone() for p in self.pools]

    def only(self, rows):
        """Only these rows have changed."""
        keep = torch.ones(self.room[0].shape[0], dtype=torch.bool, device=DEV)
        if rows:
            keep[torch.tensor(rows, device=DEV) + 2] = False
        return all(torch.equal(r[keep], b[keep]) for r, b in zip(self.room, self.before))


def run_block(w, pools, indptr, indices, positions):
    import clusterfusionplus_b200 as cf
    B = indptr.numel() - 1
    x, res = O.seeded_normal((B, H), 3, device=DEV), O.seeded_normal((B, H), 4, device=DEV)
    out, res_out = torch.empty_like(x), torch.empty_like(x)
    ptr = [torch.tensor([p.data_ptr()], dtype=torch.int64, device=DEV) for p in pools.pools]
    cf.llama_decoder_layer_batch_decode_sglang(out, res_out, x, res, w["wqkv"], w["wo"], indptr, indices, *ptr, 0, w["g"], 1e-5, positions, w["cs"])
    return x, res, out


def close_to_lists(w, pools, x, res, out, lists, positions):
    """`lists`: for every sequence the history rows that are there; a row of the pool stands in for the new token's (its content is not read)."""
    indptr, indices = [0], []
    for rows in lists:
        indices += rows + [0]
        indptr.append(len(indices))
    ref = LO.llama_attn_block_batch_fp32(x, res, w["wqkv"], w["wo"], *pools.start, ints(indptr), ints(indices), positions, w["cs"], w["g"], 1e-5)[0]
    mx, rl = O.compare(out, ref)
    assert mx <= 2e-2 and rl <= 1e-3, (mx, rl)


def test_paged_block_with_an_empty_list(cuda_device, llama):
    """A request without tokens owns no row: nothing is stored for it, least of all over the last row of the request before it."""
    pools = Pools(300)
    rows = list(range(10, 51)), list(range(100, 230))
    positions = torch.tensor([40, 0, 129], device=DEV)
    x, res, out = run_block(llama, pools, ints([0, 41, 41, 171]), ints(rows[0] + rows[1]), positions)
    assert pools.only([50, 229])
    close_to_lists(llama, pools, x, res, out, [rows[0][:-1], [], rows[1][:-1]], positions)


@pytest.mark.parametrize("batch", [1, 5, 16])
def test_paged_block_with_the_lists_of_a_plan_that_did_not_fit(cuda_device, llama, batch):
    import clusterfusionplus_b200 as cf
    pools = Pools(64)
    p = cf.paged_kv_plan(ints([16] * batch), ints([1] * batch), torch.zeros(batch, 4, dtype=torch.int32, device=DEV), ints([1]), ints([0]), 16, batch, 32 * batch)
    assert int(p.status) != 0
    x, res, out = run_block(llama, pools, p.kv_indptr.clone(), p.kv_indices.clone(), p.positions)
    assert pools.only([])
    close_to_lists(llama, pools, x, res, out, [[]] * batch, p.positions)


def test_paged_block_leaves_out_entries_below_zero(cuda_device, llama):
    """Pages that were never given: their rows are not read and not written, and the call says so."""
    import clusterfusionplus_b200 as cf
    pools = Pools(400)
    lists = [list(range(0, 200)), list(range(200, 209)), list(range(300, 340)), list(range(360, 380))]
    lists[0][3], lists[0][128:140], lists[0][199] = -1, [-1] * 12, 395          # inside a tile, across its border
    lists[1][-1] = -1                                                           # the new token's own row
    lists[2][:-1] = [-1] * 39                                                   # the whole history
    lists[3][0] = -2147483648
    positions = torch.tensor([len(x) - 1 for x in lists], device=DEV)
    starts = [0]
    for rows in lists:
        starts.append(starts[-1] + len(rows))
    x, res, out = run_block(llama, pools, ints(starts), ints(sum(lists, [])), positions)
    with pytest.raises(RuntimeError, match="status 8"):
        cf.device_status()
    assert pools.only([395, 339, 379])
    close_to_lists(llama, pools, x, res, out, [[r for r in rows[:-1] if r >= 0] for rows in lists], positions)


@pytest.mark.parametrize("batch", list(range(1, 17)))
def test_plan_goes_into_the_paged_block_as_it_is(cuda_device, llama, batch):
    """kv_indptr, kv_indices and positions of a plan, not copied, for every batch of the block; the same as from tensors of their own."""
    import clusterfusionplus_b200 as cf
    rng = random.Random(batch)
    lens = [rng.choice([0, 15, 16, rng.randint(1, 60)]) for _ in range(batch)]
    ids = list(range(5 * batch))
    rng.shuffle(ids)
    table = [[ids.pop() if i * 16 < n else -1 for i in range(4)] for n in lens]
    p = cf.paged_kv_plan(ints(lens), ints([1] * batch), ints(table), ints(ids), ints([len(ids)]), 16, batch, sum(lens) + batch + 3)
    assert int(p.status) == 0
    pools = [Pools(80 * batch) for _ in range(2)]
    *_, one = run_block(llama, pools[0], p.kv_indptr, p.kv_indices, p.positions)
    *_, two = run_block(llama, pools[1], p.kv_indptr.clone(), p.kv_indices.clone(), ints(lens).long())
    assert torch.equal(one, two) and all(torch.equal(a, b) for a, b in zip(pools[0].room, pools[1].room))
    assert pools[0].only(p.slot_map.tolist())


def test_plan_with_idle_requests_goes_into_the_paged_block(cuda_device, llama):
    """Places of a batch that hold no request: no page, no row, no position of their own in `positions`."""
    import clusterfusionplus_b200 as cf
    lens, new = [0, 31, 0, 16], [0, 1, 0, 1]
    p = cf.paged_kv_plan(ints(lens), ints(new), ints([[-1] * 3, [5, 2, -1], [-1] * 3, [0, -1, -1]]), ints([9, 7]), ints([2]), 16, 4, 64)
    assert int(p.status) == 0 and p.slot_map.tolist() == [47, 7 * 16, -1, -1]
    pools, positions = Pools(192), (p.kv_lens - 1).clamp(min=0).long()
    x, res, out = run_block(llama, pools, p.kv_indptr, p.kv_indices, positions)
    assert pools.only([47, 112])
    rows = p.kv_indices.tolist()
    close_to_lists(llama, pools, x, res, out, [[], rows[:31], [], rows[32:48]], positions)


# ------------------------------------------------------------------------------------------------------------ the free list
@pytest.mark.parametrize("count", [10, 4, 2147483647, -1])
def test_plan_refuses_a_count_that_the_list_cannot_have(cuda_device, count):
    """Two steps from a count beyond the list would deal the same pages out twice; release refuses such a count too."""
    import clusterfusionplus_b200 as cf
    table, free, n, lens = ints([[-1] * 2, [-1] * 2]), ints([9, 8, 7]), ints([count]), ints([0, 0])
    for new in ([16, 0], [0, 16], [0, 0]):
        p = cf.paged_kv_plan(lens, ints(new), table, free, n, 16, 16)
        assert int(p.status) == 1 and int(p.free_count) == count and (table == -1).all() and (p.slot_map == -1).all() and p.kv_lens.tolist() == [0, 0]
    _, status = cf.paged_kv_release(ints([0, 0]), lens, table, free, n, 16)
    assert int(status) == 1


def test_plans_of_several_steps_deal_no_page_out_twice(cuda_device):
    import clusterfusionplus_b200 as cf
    table, free, n, lens = torch.full((4, 8), -1, dtype=torch.int32, device=DEV), torch.randperm(32, device=DEV).int(), ints([32]), ints([0] * 4)
    for _ in range(8):
        p = cf.paged_kv_plan(lens, ints([16] * 4), table, free, n, 16, 64)
        assert int(p.status) == 0
        lens, n = p.kv_lens, p.free_count
    assert sorted(table.flatten().tolist()) == list(range(32)) and int(n) == 0
    p = cf.paged_kv_plan(lens, ints([0, 0, 0, 1]), table, free, n, 16, 64)
    assert int(p.status) == 1 + 2


# ----------------------------------------------------------------------------------------------------------- attention's range
@pytest.fixture(params=["by_size", "line", "prompt"])
def schedule(request, monkeypatch):
    """Clusters or what the sizes choose, the line of tiles with a workspace, 128 rows at a time on the tensor cores (a large hint asks for it)."""
    import clusterfusionplus_b200 as cf
    from clusterfusionplus_b200 import serving
    if request.param == "line":
        monkeypatch.setattr(serving, "_workspace", 64 << 20)
    if request.param == "prompt":
        plain = cf.kv4_attention
        monkeypatch.setattr(cf, "kv4_attention", lambda *a, **k: plain(*a, **(k | {"max_q_len": 4096})))


def near(got, ref):
    """rel-L2 of the roundings that the kernels are allowed (probabilities, operands and results once each): 1e-3 for fp16 results, 2.5e-3 for bf16;
    fp16 results below its normal range are off by half a step of 2^-24 besides."""
    err = (got.double().cpu() - ref).norm()
    tol = (1e-3 if got.dtype == torch.float16 else 2.5e-3) * ref.norm() + (2.0 ** -25 * math.sqrt(ref.numel()) if got.dtype == torch.float16 else 0.0)
    assert err <= tol, (err / ref.norm()).item()


def sink_case(count, T, D, dtype, gap, std, at, seed=1):
    """Rows whose token `at` stands `gap` nats above the middle of the others and has next to no value."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    base = torch.randn(2, D, device=DEV, generator=g)                                   # a direction for each cached head
    q = base.repeat_interleave(2, 0)[None] + 0.05 * torch.randn(count, 4, D, device=DEV, generator=g)
    key = torch.randn(T, 2, D, device=DEV, generator=g)
    value = torch.randn(T, 2, D, device=DEV, generator=g) * std
    key[at] = base * (gap * D ** 0.5) / (base * base).sum(-1, keepdim=True)
    value[at] *= 0.02 if gap < 12 else 0.0
    return q.to(dtype), key.to(dtype), value.to(dtype)


@pytest.mark.parametrize("dtype,std", [(torch.bfloat16, 0.005), (torch.bfloat16, 0.02), (torch.float16, 0.02), (torch.float16, 0.1)])
@pytest.mark.parametrize("gap", [0.0, 7.0, 10.0, 14.0])
@pytest.mark.parametrize("count,at", [(1, 0), (1, 1234), (6, 0), (40, 3)])
def test_attention_with_one_dominant_token_of_little_value(cuda_device, schedule, dtype, std, gap, count, at):
    """What the other tokens give has to keep its precision: small probabilities times small scales."""
    import clusterfusionplus_b200 as cf
    T, D = 2000, 128
    q, key, value = sink_case(count, T, D, dtype, gap, std, at)
    cache = cf.kv4_cache(125, 2, 16, D)
    cf.kv4_append(key, value, ints(list(range(T))), cache)
    K, V = S.unpack(cache, D)
    table = [list(range(125))]
    got = cf.kv4_attention(q, cache, ints(table), ints([T]), ints([0, count]), max_q_len=count)
    near(got, S.attention(q, K, V, table, [T], [0, count], D ** -0.5))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("count", [1, 3, 40])
def test_attention_of_values_of_all_sizes_in_one_request(cuda_device, schedule, dtype, D, count):
    """Tokens and groups whose scales differ by many binary orders, small ones first: fp16's largest among them, behind the last token too."""
    import clusterfusionplus_b200 as cf
    T = 700
    g = torch.Generator(device=DEV).manual_seed(D + count)
    q, key = (torch.randn(n, h, D, device=DEV, generator=g).to(dtype) for n, h in ((count, 4), (T + 20, 2)))
    size = torch.exp2(torch.randint(-6, 14, (T + 20, 1, 1), device=DEV, generator=g).float())
    size[:300] = 2.0 ** -6
    size[T:] = 2.0 ** 13
    value = (torch.randn(T + 20, 2, D, device=DEV, generator=g) * size).clamp(-30000, 30000).to(dtype)
    cache = cf.kv4_cache(45, 2, 16, D)
    cf.kv4_append(key, value, ints(list(range(T + 20))), cache)
    K, V = S.unpack(cache, D)
    table = [list(range(45))]
    for n in (T, 290):
        got = cf.kv4_attention(q, cache, ints(table), ints([n]), ints([0, count]), max_q_len=count)
        near(got, S.attention(q, K, V, table, [n], [0, count], D ** -0.5))


# -------------------------------------------------------------------------------------------------------- the type's largest values
def largest_rows(dtype, D):
    """Groups from 0, from the middle and from the lowest number to fp16's largest; bf16 beyond it too."""
    g = torch.Generator(device=DEV).manual_seed(D)
    top = torch.finfo(torch.float16).max
    x = torch.rand(32, 2, D, device=DEV, generator=g)
    x[:8] = x[:8] * top
    x[8:16] = (x[8:16] * 2 - 1) * top
    x[16:24] = x[16:24] * 35000 + 30000
    x[:24, :, 0::32], x[:24, :, 1::32] = top, -top
    x[:8, :, 1::32] = 0
    x[16:24, :, 1::32] = 30000
    if dtype == torch.bfloat16:
        x[24:28] = (x[24:28] * 2 - 1) * 1e38
    x[28:] = top
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [32, 80, 128])
def test_rows_of_the_largest_values_come_back_finite(cuda_device, dtype, D):
    import numpy as np

    import clusterfusionplus_b200 as cf
    x = largest_rows(dtype, D)
    cache, slots = cf.kv4_cache(2, 2, 16, D), list(range(32))
    want = cache.cpu().numpy().copy()
    for t in slots:
        S.store(want, t, x[t].float().cpu().numpy(), x[t].float().cpu().numpy())
    cf.kv4_append(x, x, ints(slots), cache)
    assert np.array_equal(cache.cpu().numpy(), want)
    ref = S.unpack(want, D)[0].transpose(1, 2).reshape(32, 2, D)
    for out in (torch.float16, torch.bfloat16):
        for got in cf.kv4_read(cache, ints(slots), D, out):
            assert got.isfinite().all() and ((got.double().cpu() - ref).abs() <= (torch.finfo(out).eps / 2 + 2.0 ** -24) * ref.abs() + 2.0 ** -25).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D", [32, 80, 128])
@pytest.mark.parametrize("count", [1, 5, 30])
def test_attention_over_the_largest_values(cuda_device, schedule, dtype, D, count):
    """The same finite values whatever the schedule; where all that a query sees is the largest number the result is it."""
    import clusterfusionplus_b200 as cf
    value = largest_rows(dtype, D)
    g = torch.Generator(device=DEV).manual_seed(count)
    q, key = torch.randn(count, 4, D, device=DEV, generator=g).to(dtype), torch.randn(32, 2, D, device=DEV, generator=g).to(dtype)
    for rows, n in ((slice(0, 32), 32), (slice(28, 32), 4)):
        cache = cf.kv4_cache(2, 2, 16, D)
        cf.kv4_append(key[rows].contiguous(), value[rows].contiguous(), ints(list(range(n))), cache)
        K, V = S.unpack(cache, D)
        m = min(count, n)
        got = cf.kv4_attention(q[:m], cache, ints([[0, 1]]), ints([n]), ints([0, m]), max_q_len=m)
        ref = S.attention(q[:m], K, V, [[0, 1]], [n], [0, m], D ** -0.5)
        assert got.isfinite().all()
        near(got, ref)


# -------------------------------------------------------------------------------------------------------------- log probabilities
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [50, 9000, 50304])
@pytest.mark.parametrize("far", [-1e31, -9e36, -9.99e36, -1e37, -3e38])
def test_logprobs_beside_the_type_s_largest(cuda_device, dtype, vocab, far):
    """Finite logits whose distance from the greatest is no fp32 number: probability 0, and nothing of the entropy."""
    import clusterfusionplus_b200 as cf
    top = torch.finfo(dtype).max
    x = torch.full((4, vocab), far, dtype=dtype, device=DEV)
    x[0, 7] = top
    x[1, 3], x[1, 40] = top, top
    x[2, ::2], x[2, 1::2] = 0.0, far
    x[3, 5:], x[3, 20] = -math.inf, top
    got = cf.token_logprobs(x, ints([7, 40, 0, 20]), 2)
    zeros = (vocab + 1) // 2
    want = torch.tensor([0.0, math.log(2), math.log(zeros), 0.0], device=DEV)
    tol = 2 * (vocab / 512 + 28) * 2.0 ** -24 * max(1.0, math.log(zeros))         # sums of equal numbers, as derived for all rows
    assert ((got.entropy - want).abs() <= tol).all() and ((got.logprobs + want).abs() <= tol).all(), (got.entropy, got.logprobs)
    assert got.top_tokens.tolist() == [[7, 0], [3, 40], [0, 2], [20, 0]]


# ------------------------------------------------------------------------------------------------ values that are not finite
@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("T,count,where", [(60, 30, [(40, 0)]), (700, 200, [(0, 3), (520, 33), (690, 70), (699, 0)]), (700, 1, [(300, 90)]), (700, 200, [(t, 5) for t in range(0, 700, 7)]),
                                           (300, 150, [(t, d) for t in range(200, 216) for d in range(0, 128, 32)])])
@pytest.mark.parametrize("D", [32, 96, 128])
def test_attention_marks_the_groups_of_values_that_are_not_finite(cuda_device, schedule, bad, T, count, where, D):
    """NaN in the group's dims for the queries that see such a token, and nothing of it for the others, wherever in tiles and pages it lies."""
    import clusterfusionplus_b200 as cf
    g = torch.Generator(device=DEV).manual_seed(T + D)
    q, key, value = (torch.randn(n, h, D, device=DEV, generator=g).half() for n, h in ((count, 4), (T, 2), (T, 2)))
    for t, d in where:
        value[t, 1, d % D] = bad
    cache = cf.kv4_cache(-(-T // 32) + 1, 2, 32, D)
    order = torch.randperm(-(-T // 32), device=DEV).int()
    at = torch.arange(T, device=DEV)
    cf.kv4_append(key, value, (order[at // 32] * 32 + at % 32).int(), cache)
    K, V = S.unpack(cache, D)
    table = [order.tolist()]
    got = cf.kv4_attention(q, cache, ints(table), ints([T]), ints([0, count]), max_q_len=count)
    ref = S.attention(q, K, V, table, [T], [0, count], D ** -0.5)
    assert torch.equal(got.isnan().cpu(), ref.isnan())
    fine = ~ref.isnan()
    near(got[fine.to(DEV)], ref[fine])


@pytest.mark.parametrize("T", [100, 700])
def test_attention_marks_them_where_a_cta_takes_several_tiles_of_rows(cuda_device, T):
    """More rows than the hint says: the same CTAs go through 128 rows after 128 rows, the marks of one are not those of the next."""
    import clusterfusionplus_b200 as cf
    D, count, B = 64, T, 2
    g = torch.Generator(device=DEV).manual_seed(T)
    q, key, value = (torch.randn(B * n, h, D, device=DEV, generator=g).half() for n, h in ((count, 16), (T, 8), (T, 8)))
    for t, h, d in ((T - 1, 0, 0), (T // 2, 1, 40), (0, 2, 5), (T + T // 3, 1, 1), (2 * T - 2, 7, 63)):
        value[t, h, d] = math.nan
    pages = -(-T // 16)
    cache = cf.kv4_cache(B * pages, 8, 16, D)
    at = torch.arange(B * T, device=DEV, dtype=torch.int32)
    cf.kv4_append(key, value, at // T * (pages * 16) + at % T, cache)
    K, V = S.unpack(cache, D)
    table = [list(range(pages)), list(range(pages, 2 * pages))]
    got = cf.kv4_attention(q, cache, ints(table), ints([T] * B), ints([0, count, 2 * count]), max_q_len=128)
    ref = S.attention(q, K, V, table, [T] * B, [0, count, 2 * count], D ** -0.5)
    assert torch.equal(got.isnan().cpu(), ref.isnan())
    fine = ~ref.isnan()
    near(got[fine.to(DEV)], ref[fine])


# ---------------------------------------------------------------------------------------------------------------------- strides
def test_strides_of_axes_with_one_entry_do_not_matter(cuda_device):
    """One token, or one head, cut out of rows that lie an odd number of elements apart."""
    import clusterfusionplus_b200 as cf
    room = torch.randn(9, 515, device=DEV).half()
    x = room[:, :512].unflatten(1, (8, 64))[:1]
    assert x.stride(0) == 515
    one_head = torch.as_strided(room, (3, 1, 64), (128, 7, 1))
    cache, same = cf.kv4_cache(1, 4, 16, 64), cf.kv4_cache(1, 4, 16, 64)
    cf.kv4_append(x[:, :4], x[:, 4:], ints([3]), cache)
    cf.kv4_append(x[:, :4].contiguous(), x[:, 4:].contiguous(), ints([3]), same)
    assert torch.equal(cache, same) and cache.any()
    table, n = ints([[0]]), ints([16])
    assert torch.equal(cf.kv4_attention(x, cache, table, n), cf.kv4_attention(x.contiguous(), cache, table, n))
    single = cf.kv4_cache(1, 1, 16, 64)
    cf.kv4_append(one_head, one_head, ints([0, 1, 2]), single)
    assert torch.equal(cf.kv4_attention(one_head, single, ints([[0]] * 3), ints([3] * 3)), cf.kv4_attention(one_head.contiguous(), single, ints([[0]] * 3), ints([3] * 3)))
    with pytest.raises(RuntimeError, match="strides"):
        cf.kv4_attention(room[:2, :512].as_strided((2, 8, 64), (515, 64, 1)), cache, ints([[0]] * 2), ints([16] * 2))


# ------------------------------------------------------------------------------------------ log probabilities, each to its own bound
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,spread", [(40, 200, 3.0), (200, 4097, 1.0), (3, 50304, 3.0), (300, 50304, 2.5), (5, 151936, 6.0)])
def test_log_probabilities_to_fp32_s_precision(cuda_device, dtype, rows, vocab, spread):
    """log p = (x - m) - log z, with u = 2^-24: x - m and the result round once each, logf is good to 2 u |log z|.  z is a sum of positive terms: runs
    of at most vocab / 512 and 12 levels of joins, which round twice and scale by ex2 (4 u) each; a term's exponent d = x - m <= 4 + log-distance
    rounds with 2.5 u |d| (difference, product, constant), whose mean under p is at most E|d| = log z - H + 4, and ex2 is good to 4 u."""
    import clusterfusionplus_b200 as cf
    g = torch.Generator(device=DEV).manual_seed(rows + vocab)
    x = (torch.randn(rows, vocab, device=DEV, generator=g) * spread).to(dtype)
    tokens = torch.randint(0, vocab, (rows,), device=DEV, generator=g)
    got = cf.token_logprobs(x, tokens, 8)
    lp, h, tl, ti = (t.to(DEV) for t in S.logprobs(x, tokens.tolist(), 8))
    log_z = -tl[:, 0]                                                                 # of the terms relative to the greatest
    u, z_err = 2.0 ** -24, vocab / 512 + 12 * 6 + 4 + 2.5 * (log_z.abs() + 4)
    assert got.top_tokens.equal(ti)
    bound = u * (z_err + 2 * (log_z.abs() + 4) + 8)                                   # the reference m may lie up to 4 below the greatest
    for a, b in ((got.logprobs[:, None], lp[:, None]), (got.top_logprobs, tl)):
        err = (a.double() - b).abs()
        assert (err <= bound[:, None] + u * 2 * b.abs()).all(), (err / bound[:, None]).max().item()
    # w / z: the same relative errors on a sum whose terms are |d| p
    err = (got.entropy.double() - h).abs()
    assert (err <= bound + u * (2 * z_err + 8) * (log_z.abs() + 4)).all(), (err / bound).max().item()


# -------------------------------------------------------------------------------------------------------------- a prompt's logits
@pytest.mark.parametrize("m,n,k", [(1, 1024, 1024), (23, 1024, 512), (130, 2056, 2560), (257, 50304, 1024)])
def test_linear_with_an_fp32_result(cuda_device, m, n, k):
    """Products of fp16 numbers are exact in fp32; a sum of k of them is off by at most k 2^-24 of the sum of their sizes."""
    from clusterfusionplus_b200._lib import CF_OUT_FP32
    from clusterfusionplus_b200.decoder import prefill_linear
    g = torch.Generator(device=DEV).manual_seed(m + n)
    x, w, b = torch.randn(m, k, device=DEV, generator=g).half(), (torch.randn(n, k, device=DEV, generator=g) * 0.3).half(), torch.randn(n, device=DEV, generator=g).half()
    for bias in (None, b):
        got = prefill_linear(x, w, bias, act=CF_OUT_FP32)
        assert got.dtype == torch.float32 and got.shape == (m, n)
        ref, size = x.double() @ w.double().t(), x.abs().double() @ w.abs().double().t()
        if bias is not None:
            ref, size = ref + bias.double(), size + bias.abs().double()
        assert ((got.double() - ref).abs() <= (k + 1) * 2.0 ** -24 * size).all()
    with pytest.raises(RuntimeError, match="residual"):
        prefill_linear(x, w, residual=torch.zeros(m, n, device=DEV, dtype=torch.float16), act=CF_OUT_FP32)


def test_score_does_not_round_its_logits(cuda_device):
    """Logits of tens, where an fp16 rounding alone is 8e-3 to 3e-2: the log probabilities of the hidden states' own logits in 64 bits."""
    import clusterfusionplus_b200 as cf
    from clusterfusionplus_b200._lib import check, lib
    mini = O.Shape("mini", hidden=512, heads=4, head_dim=128, rotary=32, ffn=2048, vocab=1024, layers=1)
    layers, head = [O.make_layer_weights(mini, 0, seed=5, device=DEV, std=0.05)], O.make_head_weights(mini, seed=5, device=DEV, std=0.05)
    head["embed_out"] = head["embed_out"] * 20
    d = cf.CfDims()
    d.hidden, d.heads, d.head_dim, d.rotary, d.ffn, d.vocab = 512, 4, 128, 32, 2048, 1024
    dec = cf.PythiaDecoder(d, layers, head, [(torch.zeros(64, 512, dtype=torch.float16, device=DEV), torch.zeros(64, 512, dtype=torch.float16, device=DEV))], 64, use_graph=False)
    rng = random.Random(3)
    tokens = [rng.randrange(1024) for _ in range(40)]
    got = dec.score(tokens, 3)
    x, y, w = dec._ingest(tokens)[1], torch.empty(39, 512, dtype=torch.float16, device=DEV), head
    check(lib.cf_prefill_layernorm2(x.data_ptr(), w["final_ln_weight"].data_ptr(), w["final_ln_bias"].data_ptr(), None, None, y.data_ptr(), None, 39, 512, 1e-5,
                                    torch.cuda.current_stream().cuda_stream))
    lg = y.double() @ w["embed_out"].double().t()
    assert 32 < lg.abs().amax() < 128
    lp, h, tl, _ = S.logprobs(lg, tokens[1:], 3)
    # a logit is a sum in fp32, in 32 steps of 16 products: each cuts off less than 2^-23 of a partial sum below 128, 5e-4 in all; a log probability takes
    # two of them, the entropy one for each |log p| <= 1 that p spreads over
    for a, b in ((got.logprobs, lp), (got.top_logprobs, tl), (got.entropy, h)):
        assert (a.double().cpu() - b).abs().max() <= 1e-3
    dec.close()


# ------------------------------------------------------------------------------------------------------- few rows: 32-bit precision
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("way", [None, 64 << 20])
@pytest.mark.parametrize("D", [64, 80, 128])
@pytest.mark.parametrize("T,count", [(24, 1), (500, 1), (500, 3), (3000, 8)])
def test_attention_of_few_rows_rounds_only_its_result(cuda_device, monkeypatch, dtype, way, D, T, count):
    """Codes, keys and values are exact operands, probabilities keep 22 bits: what is left are fp32 sums (2^-16 of the largest value, as for all schedules)
    and the result's rounding."""
    import clusterfusionplus_b200 as cf
    from clusterfusionplus_b200 import serving
    monkeypatch.setattr(serving, "_workspace", way)
    g = torch.Generator(device=DEV).manual_seed(T + D)
    q, key, value = (torch.randn(n, h, D, device=DEV, generator=g).to(dtype) for n, h in ((count, 4), (T, 2), (T, 2)))
    cache = cf.kv4_cache(-(-T // 16), 2, 16, D)
    cf.kv4_append(key, value, ints(list(range(T))), cache)
    K, V = S.unpack(cache, D)
    table = [list(range(-(-T // 16)))]
    got = cf.kv4_attention(q, cache, ints(table), ints([T]), ints([0, count]), max_q_len=count)
    ref = S.attention(q, K, V, table, [T], [0, count], D ** -0.5)
    off = (got.double().cpu() - ref).abs() - torch.finfo(dtype).eps / 2 * ref.abs() - 2.0 ** -25
    assert (off <= 2.0 ** -16 * V.abs().amax()).all(), (off / V.abs().amax()).max().item()


@pytest.mark.parametrize("n", [0, 1, 3])
def test_attention_of_a_mixed_step_in_two_calls(cuda_device, n):
    """Decoding requests and prompt chunks of one step: parts of the same lists, the columns in use of a wide table, and one output."""
    import clusterfusionplus_b200 as cf
    lens, counts, D = [300, 17, 64, 200, 90], [1] * n + [150, 80], 64
    lens = lens[:n] + lens[3:]
    g = torch.Generator(device=DEV).manual_seed(n)
    starts = [0]
    for c in counts:
        starts.append(starts[-1] + c)
    q = torch.randn(starts[-1] + 4, 8, D, device=DEV, generator=g).half()
    T = sum(-(-x // 16) * 16 for x in lens)
    key, value = (torch.randn(T, 2, D, device=DEV, generator=g).half() for _ in range(2))
    cache, table, at = cf.kv4_cache(T // 16, 2, 16, D), [], 0
    cf.kv4_append(key, value, ints(list(range(T))), cache)
    for x in lens:
        table.append(list(range(at, at + -(-x // 16))) + [-1] * (1000 - -(-x // 16)))
        at += -(-x // 16)
    out, t, kv, ip = torch.full_like(q, 7.0), ints(table), ints(lens), ints(starts)
    if n:
        cf.kv4_attention(q, cache, t[:n, :19], kv[:n], ip[:n + 1], out=out)
        assert (out[n:] == 7).all()
    cf.kv4_attention(q, cache, t[n:, :19], kv[n:], ip[n:], max_q_len=150, out=out)
    assert (out[starts[-1]:] == 7).all()
    K, V = S.unpack(cache, D)
    near(out[:starts[-1]], S.attention(q[:starts[-1]], K, V, table, lens, starts, D ** -0.5))


@pytest.mark.parametrize("D,heads,kv_heads,B,T,rows", [(64, 2, 2, 256, 16384, 1), (128, 4, 1, 600, 8192, 3), (128, 2, 2, 150, 4096, 1), (64, 1, 1, 1, 200000, 1)])
@pytest.mark.parametrize("way", ["rule", "no workspace"])
@pytest.mark.parametrize("size", [0.05, 1.0])
def test_attention_of_long_requests_in_a_full_batch(cuda_device, monkeypatch, D, heads, kv_heads, B, T, rows, way, size):
    """Hundreds of tiles for each warp, next to even probabilities: the sums are a few hundred times the result, and cutting off each of their steps must
    not show in it.  All requests name the same pages."""
    import clusterfusionplus_b200 as cf
    from clusterfusionplus_b200 import serving
    if way == "no workspace":
        monkeypatch.setattr(serving, "_workspace", 0)
    g = torch.Generator(device=DEV).manual_seed(T + B)
    key, value = (torch.randn(T, kv_heads, D, device=DEV, generator=g).half() for _ in range(2))
    q = (torch.randn(B * rows, heads, D, device=DEV, generator=g) * size).half()
    cache = cf.kv4_cache(-(-T // 64), kv_heads, 64, D)
    cf.kv4_append(key, value, torch.arange(T, device=DEV, dtype=torch.int32), cache)
    table = torch.arange(-(-T // 64), device=DEV, dtype=torch.int32)[None].repeat(B, 1)
    got = cf.kv4_attention(q, cache, table, ints([T] * B), ints([rows * b for b in range(B + 1)]), max_q_len=rows)
    K, V = S.unpack(cache, D)
    for b in {0, B // 3, B - 1}:
        at = slice(b * rows, (b + 1) * rows)
        near(got[at], S.attention(q[at], K, V, [list(range(-(-T // 64)))], [T], [0, rows], D ** -0.5))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("rows", [1, 5, 40])
def test_attention_of_queries_that_are_not_finite(cuda_device, schedule, bad, rows):
    """They make their own row and head NaN; every other result keeps its bits."""
    import clusterfusionplus_b200 as cf
    g = torch.Generator(device=DEV).manual_seed(rows)
    key, value = (torch.randn(600, 2, 64, device=DEV, generator=g).half() for _ in range(2))
    cache, table, lens, starts = cf.kv4_cache(38, 2, 16, 64), ints([list(range(38))]), ints([600]), ints([0, rows])
    cf.kv4_append(key, value, ints(list(range(600))), cache)
    q = torch.randn(rows, 8, 64, device=DEV, generator=g).half()
    want = cf.kv4_attention(q, cache, table, lens, starts, max_q_len=rows)
    q[rows // 2, 3, 7] = bad
    got = cf.kv4_attention(q, cache, table, lens, starts, max_q_len=rows)
    assert got[rows // 2, 3].isnan().all()
    same = got == want
    same[rows // 2, 3] = True
    assert same.all()
