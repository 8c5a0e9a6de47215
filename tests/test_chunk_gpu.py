"""The chunked path over the paged cache on the device: plan (block tables, slot maps), append by slots, causal and
windowed attention of packed chunks, each against a plain restatement, and a run of them together.

Attention tolerances, per element, from the roundings a row goes through.  With e = half a step of the 16-bit type
(bf16 2^-8, fp16 2^-11 relative) and A = sum w |v| (the oracle's second result): the weights enter the P V product
rounded to the type, at most e * A; the exponentials themselves and their fp32 sum are good to 2^-13 relative, at most
2 * 2^-13 * A with the normalisation; fp16 weights below the normal range are off by 2^-25 of the largest weight each,
at most rows * 2^-25 * max|v|; the output is rounded once, e * |o|.  Scores are fp32 dot products of 16-bit values of
magnitude about 1: their error is below 128 * 2^-24 * 12 = 2^-13.4 absolute for the unit-variance inputs used here, and
so that of a weight, relative, once more 2^-13 * 2 * A.
"""
import pytest
import torch

from oracle import attention_oracle as ao
from subspec_b200.attention import append_paged_kv_slots, chunk_attention_paged, tree_attention_paged, window_attention_paged
from subspec_b200.pages import DevicePagePool
from subspec_b200.step import SpeculativeLoopBatch

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------- plan

class _Pages:
    """The page lists in Python: lowest free page first, requests in order, releases before allocations."""

    def __init__(self, batch, num_pages, page_len):
        self.page_len, self.free = page_len, set(range(num_pages))
        self.pages, self.kv_len = [[] for _ in range(batch)], [0] * batch

    def plan(self, n_new, set_len=None):
        base = list(self.kv_len if set_len is None else set_len)
        for b, rows in enumerate(base):
            keep = -(-rows // self.page_len)
            self.free.update(self.pages[b][keep:])
            self.pages[b] = self.pages[b][:keep]
        indptr, slots, positions, requests = [0], [], [], []
        for b, (rows, n) in enumerate(zip(base, n_new)):
            self.kv_len[b] = rows + n
            while len(self.pages[b]) * self.page_len < rows + n:
                page = min(self.free)
                self.free.remove(page)
                self.pages[b].append(page)
            for p in range(rows, rows + n):
                slots.append(self.pages[b][p // self.page_len] * self.page_len + p % self.page_len)
                positions.append(p)
                requests.append(b)
            indptr.append(indptr[-1] + n)
        return indptr, slots, positions, requests


def _check_plan(pool, want, plan, expected):
    indptr, slots, positions, requests = expected
    T, pad = indptr[-1], pool.max_append - indptr[-1]
    assert plan.q_indptr.tolist() == indptr
    assert plan.slot_map.tolist() == slots + [-1] * pad
    assert plan.positions.tolist() == positions + [0] * pad
    assert plan.batch_indices.tolist() == requests + [-1] * pad
    assert plan.kv_len.tolist() == want.kv_len
    assert pool.n_pages.tolist() == [len(p) for p in want.pages]
    width = pool.pages_per_seq
    assert plan.page_table.tolist() == [p + [-1] * (width - len(p)) for p in want.pages]
    assert pool.kv_last_page_len.tolist() == [(n - 1) % pool.page_len + 1 if n else 0 for n in want.kv_len]
    assert pool.num_free_pages() == len(want.free)
    pool.check_status()


@pytest.mark.parametrize("batch,num_pages,page_len,steps,seed", [
    (1, 1, 1, 3, 0), (1, 33, 16, 4, 1), (3, 64, 5, 6, 2), (7, 200, 16, 6, 3), (40, 1000, 8, 5, 4), (130, 3100, 3, 4, 5),
    (300, 9000, 16, 3, 6)])
def test_plan_follows_the_page_lists(cuda_lib, batch, num_pages, page_len, steps, seed):
    """Scripted steps: prompts, single tokens, requests that bring nothing, finish (0 rows kept) or are cut back;
    batches above and below a warp, a CTA's requests and a cluster; page counts that end inside a mask word."""
    g = torch.Generator().manual_seed(seed)
    r = lambda hi: int(torch.randint(0, hi + 1, (1,), generator=g))
    room = num_pages // batch * page_len  # rows a request may hold so that the pages never run out
    want = _Pages(batch, num_pages, page_len)
    pool = DevicePagePool(batch, num_pages, page_len, max(1, num_pages // batch), DEV, max_append=batch * room + 3)
    for step in range(steps):
        base = None
        if step % 2:
            base = [r(n) if r(2) else (0 if r(3) == 0 else n) for n in want.kv_len]
        rows = want.kv_len if base is None else base
        n_new = [min(room - x, [0, 1, r(room)][r(2)]) for x in rows]
        expected = want.plan(n_new, base)
        plan = pool.plan_chunks(_i32(n_new), set_len=None if base is None else _i32(base))
        _check_plan(pool, want, plan, expected)


def test_plan_and_tree_steps_share_the_pool(cuda_lib):
    """A chunk, a tree step through `update`, the cut back to what was kept, another chunk: one set of page lists."""
    want, pool = _Pages(2, 40, 4), DevicePagePool(2, 40, 4, 20, DEV, max_append=64)
    _check_plan(pool, want, pool.plan_chunks(_i32([9, 6])), want.plan([9, 6]))
    pool.update(add_all=8, mode="tree", tree_tokens=8)
    want.plan([8, 8])
    assert pool.n_pages.tolist() == [len(p) for p in want.pages]
    _check_plan(pool, want, pool.plan_chunks(_i32([0, 30]), set_len=_i32([11, 7])), want.plan([0, 30], [11, 7]))


def test_plan_reports_what_does_not_fit(cuda_lib):
    pool = DevicePagePool(2, 5, 4, 4, DEV, max_append=40)
    plan = pool.plan_chunks(_i32([16, 8]))                 # four pages and two of five
    assert pool.n_pages.tolist() == [4, 1] and plan.slot_map[20:].tolist() == [-1] * 20
    with pytest.raises(ValueError, match="page"):
        pool.check_status()
    pool = DevicePagePool(1, 50, 4, 3, DEV, max_append=40)
    plan = pool.plan_chunks(_i32([15]))                    # four pages, the list holds three
    assert plan.kv_len.tolist() == [12] and plan.slot_map[12:15].tolist() == [-1] * 3 and plan.slot_map[11].item() == 11
    with pytest.raises(ValueError, match="page"):
        pool.check_status()
    pool = DevicePagePool(2, 50, 4, 3, DEV, max_append=4)
    plan = pool.plan_chunks(_i32([3, 3]))                  # six tokens, room for four
    assert plan.q_indptr.tolist() == [0, 3, 6] and plan.slot_map.tolist() == [0, 1, 2, 4]
    with pytest.raises(ValueError, match="count"):
        pool.check_status()
    plan = pool.plan_chunks(_i32([-2, 1]))                 # a negative length counts as none
    assert plan.kv_len.tolist() == [3, 4]
    with pytest.raises(ValueError, match="count"):
        pool.check_status()
    huge = pool.plan_chunks(_i32([2 ** 31 - 1, 2 ** 31 - 1]))
    assert huge.kv_len.tolist() == [12, 12]
    with pytest.raises(ValueError):
        pool.check_status()


# ---------------------------------------------------------------- append

@pytest.mark.parametrize("T,H,D,page_len,dtype", [
    (1, 1, 64, 1, torch.bfloat16), (7, 2, 128, 16, torch.float16), (333, 4, 128, 5, torch.bfloat16),
    (1000, 8, 64, 32, torch.float16), (64, 3, 40, 16, torch.bfloat16), (5, 1, 8, 3, torch.float16)])
def test_append_by_slots(cuda_lib, T, H, D, page_len, dtype):
    """Rows land bit for bit (NaN and all), nothing else moves; k and v as slices of a fused projection."""
    g = torch.Generator().manual_seed(T)
    P = T // page_len + 4
    pool = torch.randn(2, P, 2, page_len, H, D, generator=g).to(dtype)
    qkv = torch.randn(T, 3 * H, D, generator=g).to(dtype)
    qkv[0, H, 0] = float("nan")
    slots = torch.randperm(P * page_len, generator=g)[:T]
    if T > 3:
        slots[1] = -1
    got, dq = pool.to(DEV), qkv.to(DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    append_paged_kv_slots(got, 1, dq[:, H:2 * H], dq[:, 2 * H:], slot_map=slots.to(DEV), status=status)
    for t, s in enumerate(slots.tolist()):
        if s >= 0:
            pool[1, s // page_len, 0, s % page_len] = qkv[t, H:2 * H]
            pool[1, s // page_len, 1, s % page_len] = qkv[t, 2 * H:]
    assert torch.equal(got.cpu().view(torch.int16), pool.view(torch.int16)) and status.item() == 0


def test_append_layouts_and_bad_slots(cuda_lib):
    """Rows at odd addresses and heads-first strides are taken too; a slot past the pool is skipped and reported."""
    pool = torch.zeros(1, 4, 2, 4, 2, 64, dtype=torch.bfloat16, device=DEV)
    flat = torch.arange(1, 2 * 3 * 64 + 2, device=DEV).to(torch.bfloat16)
    k = flat[1:].view(2, 3, 64).transpose(0, 1)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    append_paged_kv_slots(pool, 0, k, k + 1, slot_map=torch.tensor([15, 16, 2 ** 40], device=DEV), status=status)
    assert torch.equal(pool[0, 3, 0, 3], k[0]) and torch.equal(pool[0, 3, 1, 3], (k + 1)[0])
    assert int((pool != 0).sum()) == 2 * 2 * 64 and status.item() != 0


# ---------------------------------------------------------------- attention

def _setup(seed, new, cached, heads, kv_heads, D=128, page_len=16, dtype=torch.bfloat16, layers=2, layer=1, stale="nan",
           pad=0):
    """A cache with pages in no order; rows that hold nothing (and, `stale`, whole pages) are NaN."""
    g = torch.Generator().manual_seed(seed)
    B = len(new)
    total = [n + c for n, c in zip(new, cached)]
    width = max(1, max(-(-t // page_len) for t in total) + 1)
    P = sum(-(-t // page_len) for t in total) + 3
    order = torch.randperm(P, generator=g).tolist()
    pool = torch.full((layers, P, 2, page_len, kv_heads, D), float("nan") if stale == "nan" else 7.0).to(dtype)
    table = torch.full((B, width), -1, dtype=torch.int32)
    ks, vs = [], []
    for b, t in enumerate(total):
        k, v = torch.randn(t, kv_heads, D, generator=g).to(dtype), torch.randn(t, kv_heads, D, generator=g).to(dtype)
        for j in range(-(-t // page_len)):
            page = order.pop()
            table[b, j] = page
            rows = k[j * page_len:(j + 1) * page_len]
            pool[layer, page, 0, :len(rows)] = rows
            pool[layer, page, 1, :len(rows)] = v[j * page_len:(j + 1) * page_len]
        ks.append(k)
        vs.append(v)
    q = torch.randn(sum(new) + pad, heads, D, generator=g).to(dtype)
    indptr = [sum(new[:b]) for b in range(B + 1)]
    return dict(q=q, pool=pool, table=table, ks=ks, vs=vs, kv_len=total, indptr=indptr, layer=layer, new=new)


def _run(c, window=0, sinks=0, status=None, **kw):
    args = dict(page_table=c["table"].to(DEV), kv_len=_i32(c["kv_len"]), q_indptr=_i32(c["indptr"]), status=status, **kw)
    if window:
        return window_attention_paged(c["q"].to(DEV), c["pool"].to(DEV), c["layer"], window=window, sinks=sinks, **args)
    return chunk_attention_paged(c["q"].to(DEV), c["pool"].to(DEV), c["layer"], **args)


def _tolerance(o, mag, rows, dtype, vmax):
    e = torch.finfo(dtype).eps / 2
    return e * o.abs() + (e + 4 * 2 ** -13) * mag + rows * 2 ** -25 * vmax + 1e-6


def _check(c, got, window=0, sinks=0, only=None):
    for b, n in enumerate(c["new"]):
        if n == 0 or (only is not None and b not in only):
            continue
        lo = c["indptr"][b]
        want, mag = ao.chunk_attention(c["q"][lo:lo + n], c["ks"][b], c["vs"][b], window, sinks)
        err = (got[lo:lo + n].double().cpu() - want).abs()
        tol = _tolerance(want, mag, c["kv_len"][b], c["q"].dtype, 6.0)
        assert bool((err <= tol).all()), (b, float((err - tol).max()), int((~(err <= tol)).sum()))


def _run_and_check(c, window=0, sinks=0, **kw):
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    got = _run(c, window, sinks, status, **kw)
    assert status.item() == 0
    _check(c, got, window, sinks)
    return got


LAYOUTS = [(1, 1), (4, 4), (28, 4), (8, 1), (6, 2), (32, 8)]


@pytest.mark.parametrize("heads,kv_heads", LAYOUTS)
@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.float16)])
def test_single_tokens(cuda_lib, heads, kv_heads, D, dtype):
    """Decode steps: caches from nothing to several tiles, lengths one off the tile and page borders."""
    cached = [0, 1, 15, 16, 126, 127, 128, 400, 255, 63]
    c = _setup(1, [1] * len(cached), cached, heads, kv_heads, D=D, dtype=dtype)
    _run_and_check(c, max_q_len=1)
    _run_and_check(c)


@pytest.mark.parametrize("heads,kv_heads", LAYOUTS)
@pytest.mark.parametrize("D,dtype", [(128, torch.float16), (64, torch.bfloat16), (128, torch.bfloat16)])
def test_chunks(cuda_lib, heads, kv_heads, D, dtype):
    """Ragged chunks, requests that bring nothing, prompts without a cache, rows that end inside every tile size."""
    c = _setup(2, [37, 0, 1, 130, 5], [300, 20, 0, 0, 129], heads, kv_heads, D=D, dtype=dtype)
    _run_and_check(c)
    _run_and_check(c, max_q_len=130)


@pytest.mark.parametrize("page_len", [1, 3, 4, 8, 24, 40, 64, 96, 128, 192, 256, 1024])
def test_page_lengths(cuda_lib, page_len):
    c = _setup(3, [70, 1, 9], [200, 300, 0], 4, 2, page_len=page_len)
    _run_and_check(c)
    _run_and_check(c, 50, 3)
    c = _setup(4, [1, 1, 2], [200, 129, 0], 4, 2, page_len=page_len, D=64)
    _run_and_check(c, max_q_len=2)
    _run_and_check(c, 50, 3, max_q_len=2)


@pytest.mark.parametrize("new,cached", [
    ([1], [9000]), ([1, 1, 1], [3000, 40, 0]), ([3], [5000]), ([60, 3], [2700, 90]), ([300], [4000]), ([9, 1, 200], [64, 3000, 1500])])
@pytest.mark.parametrize("heads,kv_heads", [(14, 2), (4, 1)])
def test_caches_cut_into_runs(cuda_lib, new, cached, heads, kv_heads):
    """Few requests behind long caches: their cache rows are shared between many CTAs and joined."""
    c = _setup(5, new, cached, heads, kv_heads)
    _run_and_check(c)
    _run_and_check(c, 1300, 5)
    _run_and_check(c, max_q_len=max(new))


def test_many_requests(cuda_lib):
    """More requests than a warp has lanes and than are summed side by side; ones that bring nothing among them."""
    new = [[0, 1, 2, 7, 40, 0, 1, 19][i % 8] for i in range(150)]
    cached = [(37 * i) % 300 for i in range(150)]
    c = _setup(19, new, cached, 4, 1, D=64)
    _run_and_check(c)
    _run_and_check(c, 60, 3)
    c = _setup(20, [min(n, 1) for n in new], cached, 8, 1)
    _run_and_check(c, max_q_len=1)


WINDOWS = [(1, 0), (1, 1), (2, 300), (16, 0), (100, 4), (128, 128), (129, 130), (5000, 7)]


@pytest.mark.parametrize("window,sinks", WINDOWS)
def test_windows(cuda_lib, window, sinks):
    """Windows of one row, of tile lengths, longer than the cache; sinks inside, next to and over the window."""
    c = _setup(6, [1, 1, 1, 1], [0, 130, 513, 300], 8, 2)
    _run_and_check(c, window, sinks, max_q_len=1)
    c = _setup(7, [45, 260, 1], [400, 0, 310], 7, 1, dtype=torch.float16)
    _run_and_check(c, window, sinks)


def test_pages_behind_the_window_may_be_gone(cuda_lib):
    """A request that gave back the pages no token sees: their entries are -1, nothing is reported."""
    for new, window, sinks in (([1], 100, 5), ([30], 64, 0), ([200], 33, 17)):
        c = _setup(8, new, [700], 4, 2)
        first = 700 - window + 1  # lowest row of the first token's window
        for j in range(c["table"].shape[1]):
            if j * 16 >= sinks and (j + 1) * 16 <= first:
                c["table"][0, j] = -1
        _run_and_check(c, window, sinks)
        _run_and_check(c, window, sinks, max_q_len=new[0])


@pytest.mark.parametrize("new", [[1, 1], [3, 2], [90, 40], [300, 1]])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_hidden_rows_have_no_influence(cuda_lib, new, bad):
    """NaN and infinities in K and V rows that a token does not see: later rows of its own chunk, rows in front of its
    window.  The rows that do see them come out as the formula gives them."""
    c = _setup(9, new, [200, 150], 4, 2)
    for b, n in enumerate(new):
        j = c["kv_len"][b] - 1  # the last token's own row
        for rows, plane, d in ((c["vs"][b], 1, 3), (c["ks"][b], 0, 5)):
            rows[j, :, d] = bad
            c["pool"][1, c["table"][b, j // 16], plane, j % 16, :, d] = bad
    got = _run(c).float().cpu()
    for b, n in enumerate(new):
        lo = c["indptr"][b]
        want, mag = ao.chunk_attention(c["q"][lo:lo + n], c["ks"][b], c["vs"][b])
        w, g = want[:n - 1], got[lo:lo + n - 1].double()
        assert bool(torch.isfinite(w).all())
        assert bool(((g - w).abs() <= _tolerance(w, mag[:n - 1], c["kv_len"][b], torch.bfloat16, 6.0)).all())
        assert torch.equal(torch.isfinite(got[lo + n - 1]), torch.isfinite(want[n - 1]))
    c = _setup(10, new, [200, 150], 4, 2)
    for b, n in enumerate(new):
        for j in range(10, 100):
            c["vs"][b][j] = c["ks"][b][j] = bad
            c["pool"][1, c["table"][b, j // 16], :, j % 16] = bad
    for kw in (dict(), dict(max_q_len=max(new)), dict(max_q_len=512)):
        got = _run(c, 50, 10, **kw).float().cpu()
        for b, n in enumerate(new):
            lo, first = c["indptr"][b], [200, 150][b]
            seen = [i for i in range(n) if first + i - 50 >= 99]  # rows whose window begins behind the bad ones
            want, mag = ao.chunk_attention(c["q"][lo:lo + n], c["ks"][b], c["vs"][b], 50, 10)
            w, g = want[seen], got[lo:lo + n][seen].double()
            assert bool(torch.isfinite(w).all()) and len(seen) == n
            assert bool(((g - w).abs() <= _tolerance(w, mag[seen], c["kv_len"][b], torch.bfloat16, 6.0)).all())


def test_scores_of_all_sizes(cuda_lib):
    """Scores that grow by hundreds along the row (the running maximum moves at every tile), scores that are all
    equal, and a scale of the caller's."""
    for new in ([1, 1], [70, 200]):
        c = _setup(11, new, [500, 300], 4, 2)
        ramp = torch.linspace(0, 30, 500 + new[0])
        c["ks"][0] *= 0
        c["ks"][0][:, :, 0] = ramp[:, None].to(torch.bfloat16)
        c["ks"][1] *= 0
        c["q"][:, :, 0] = 8.0
        for b in range(2):
            for j in range(c["kv_len"][b]):
                c["pool"][1, c["table"][b, j // 16], 0, j % 16] = c["ks"][b][j]
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        got = _run(c, status=status, sm_scale=1.5)
        for b, n in enumerate(new):
            lo = c["indptr"][b]
            want, mag = ao.chunk_attention(c["q"][lo:lo + n], c["ks"][b], c["vs"][b], sm_scale=1.5)
            # scores up to 8 * 30 * 1.5 = 360: an fp32 score is off by half a step there, 2^-16 relative in the weight
            tol = _tolerance(want, mag, c["kv_len"][b], torch.bfloat16, 6.0) + 2 ** -13 * mag
            assert bool(((got[lo:lo + n].double().cpu() - want).abs() <= tol).all()), (new, b)
        assert status.item() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("step", [4.0, 30.0, 45.0, 80.0])
def test_scores_that_rise_by_steps(cuda_lib, dtype, step):
    """Scores that rise by `step` every 100 rows, and fall again: the reference point of the weights has to follow over
    many tiles (4: it need not; 30, 45: between the tiles; 80: further than the types' weights reach within one)."""
    for new, cached in (([1], [900]), ([40], [860])):
        c = _setup(21, new, cached, 4, 2, dtype=dtype)
        n = c["kv_len"][0]
        level = (torch.arange(n) // 100).clamp(max=6) * step
        level[700:] = 0
        c["ks"][0] *= 0
        c["ks"][0][:, :, 0] = (level / 16)[:, None].to(dtype)
        c["q"] *= 0
        c["q"][:, :, 0] = 16.0
        for j in range(n):
            c["pool"][1, c["table"][0, j // 16], 0, j % 16] = c["ks"][0][j]
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        got = _run(c, status=status, sm_scale=1.0)
        want, mag = ao.chunk_attention(c["q"], c["ks"][0], c["vs"][0], sm_scale=1.0)
        # the scores are single products, exact in fp32; scaled to powers of two (up to 480 * 1.44) they are off by 2^-15
        tol = _tolerance(want, mag, n, dtype, 6.0) + 2 ** -14 * mag
        assert bool(((got.double().cpu() - want).abs() <= tol).all()) and status.item() == 0


def test_values_that_are_not_finite_and_seen(cuda_lib):
    """NaN and infinite scores and values that a row does see: the row comes out as the formula has it."""
    for new in ([1, 1], [70, 30]):
        for plane, bad in ((0, float("nan")), (1, float("nan")), (1, float("inf"))):
            c = _setup(22, new, [300, 200], 4, 2)
            for b in range(2):
                j = 133
                (c["ks"] if plane == 0 else c["vs"])[b][j, :, 7] = bad
                c["pool"][1, c["table"][b, j // 16], plane, j % 16, :, 7] = bad
            got = _run(c).double().cpu()
            for b, n in enumerate(new):
                lo = c["indptr"][b]
                want, mag = ao.chunk_attention(c["q"][lo:lo + n], c["ks"][b], c["vs"][b])
                g, fine = got[lo:lo + n], torch.isfinite(want)
                assert torch.equal(torch.isnan(g), torch.isnan(want)) and torch.equal(torch.isfinite(g), fine)
                tol = _tolerance(want, mag, c["kv_len"][b], torch.bfloat16, 6.0)
                assert bool(((g - want).abs()[fine] <= tol[fine]).all())


def test_layouts_of_q_and_out(cuda_lib):
    """q as a slice of a fused projection, heads in front of tokens, odd addresses; out with strides of its own, its
    padding and the rows behind the last request untouched."""
    c = _setup(12, [40, 3], [100, 60], 4, 2, pad=9)
    T = 52
    plan = dict(page_table=c["table"].to(DEV), kv_len=_i32(c["kv_len"]), q_indptr=_i32(c["indptr"]))
    pool, q = c["pool"].to(DEV), c["q"].to(DEV)
    fused = torch.zeros(T, 10, 128, dtype=torch.bfloat16, device=DEV)
    fused[:, 3:7] = q
    first = torch.zeros(4, T, 128, dtype=torch.bfloat16, device=DEV)
    first.copy_(q.transpose(0, 1))
    odd = torch.zeros(T * 4 * 128 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(T, 4, 128)
    odd.copy_(q)
    for x in (fused[:, 3:7], first.transpose(0, 1), odd):
        out = torch.full((4, T + 1, 136), 5.0, dtype=torch.bfloat16, device=DEV)
        view = out.transpose(0, 1)[:T, :, :128]
        assert chunk_attention_paged(x, pool, 1, out=view, **plan) is view
        _check(c, view)
        assert bool((out[:, 43:] == 5).all()) and bool((out[:, :, 128:] == 5).all())


def test_bad_lengths_and_pages_are_reported(cuda_lib):
    """A cache shorter than its new rows (tokens in front of row 0 see nothing: zeros), a length past the table, more
    tokens than `max_q_len`, page ids outside the pool."""
    for new in ([5, 2], [3, 2]):
        c = _setup(13, new, [30, 40], 4, 2)
        c["kv_len"][0] = 2
        c["ks"][0], c["vs"][0] = c["ks"][0][:2], c["vs"][0][:2]
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        got = _run(c, status=status)
        assert status.item() == 256
        _check(c, got)
        c["kv_len"][0] = 10 ** 6
        status.zero_()
        got = _run(c, status=status)
        assert status.item() != 0
        _check(c, got, only=[1])
        c["kv_len"][0] = 30
        c["indptr"] = [0, new[0], new[0] + 2]
        status.zero_()
        _run(c, status=status, max_q_len=new[0] - 1)
        assert status.item() == 256
    for new in ([1, 1], [40, 40]):
        c = _setup(14, new, [60, 60], 4, 2)
        for page in (-1, 10 ** 6):
            c["table"][0, 1] = page
            status = torch.zeros(1, dtype=torch.int32, device=DEV)
            got = _run(c, status=status)
            assert status.item() == 8
            _check(c, got, only=[1])


@pytest.mark.parametrize("seed", range(24))
def test_random_shapes(cuda_lib, seed):
    g = torch.Generator().manual_seed(500 + seed)
    r = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))
    B = r(1, 5)
    kv_heads = [1, 2, 3, 4][r(0, 3)]
    heads = kv_heads * [1, 2, 4, 5, 7, 8, 16][r(0, 6)]
    most = [1, 2, 4, 20, 90, 200][r(0, 5)]
    new, cached = [r(0, most) for _ in range(B)], [r(0, 800) for _ in range(B)]
    new[r(0, B - 1)] = most
    c = _setup(900 + seed, new, cached, heads, kv_heads, D=[64, 128][r(0, 1)], page_len=[1, 8, 16, 16, 20, 32, 64, 256][r(0, 7)],
               dtype=[torch.bfloat16, torch.float16][r(0, 1)])
    window = [0, 0, r(1, 900)][r(0, 2)]
    _run_and_check(c, window, r(0, 40) if window else 0, max_q_len=[None, most][r(0, 1)])


def test_results_do_not_depend_on_the_run(cuda_lib):
    """The same call twice, and next to another on a second stream: the same bits."""
    c = _setup(15, [1] * 20 + [150], [300 + 41 * i for i in range(20)] + [99], 28, 4)
    plan = dict(page_table=c["table"].to(DEV), kv_len=_i32(c["kv_len"]), q_indptr=_i32(c["indptr"]))
    q, pool = c["q"].to(DEV), c["pool"].to(DEV)
    a = chunk_attention_paged(q, pool, 1, **plan)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(3):
        with torch.cuda.stream(side):
            x = chunk_attention_paged(q, pool, 1, **plan)
        y = window_attention_paged(q, pool, 1, window=100, sinks=4, **plan)
        outs.append((x, y))
    torch.cuda.synchronize()
    for x, y in outs:
        assert torch.equal(x, a) and torch.equal(y, outs[0][1])


def test_captured_steps(cuda_lib):
    """Plan, append and attention captured once, replayed with other lengths: the graph reads them from the device.  A
    second graph of the same calls lives beside it."""
    H, HQ, D, page_len, B, cap = 2, 8, 128, 16, 3, 40
    g = torch.Generator().manual_seed(16)
    pages = DevicePagePool(B, 64, page_len, 16, DEV, max_append=cap)
    pool = torch.full((1, 64, 2, page_len, H, D), float("nan"), dtype=torch.bfloat16, device=DEV)
    n_new, keep = _i32([0] * B), _i32([0] * B)
    qkv = torch.zeros(cap, HQ + 2 * H, D, dtype=torch.bfloat16, device=DEV)
    out, wout = torch.zeros(cap, HQ, D, dtype=torch.bfloat16, device=DEV), torch.zeros(cap, HQ, D, dtype=torch.bfloat16, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)

    def step():
        plan = pages.plan_chunks(n_new, set_len=keep)
        append_paged_kv_slots(pool, 0, qkv[:, HQ:HQ + H], qkv[:, HQ + H:], slot_map=plan.slot_map, status=status)
        kw = dict(page_table=plan.page_table, kv_len=plan.kv_len, q_indptr=plan.q_indptr, status=status)
        chunk_attention_paged(qkv[:, :HQ], pool, 0, out=out, **kw)
        window_attention_paged(qkv[:, :HQ], pool, 0, window=20, sinks=2, out=wout, **kw)

    step()  # lazily loaded kernels
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        graphs.append(graph)
    ks, vs = [torch.zeros(0, H, D)] * B, [torch.zeros(0, H, D)] * B
    for i, new in enumerate([[12, 0, 20], [1, 1, 1], [0, 0, 0], [5, 30, 1], [1, 1, 1]]):
        rows = torch.randn(cap, HQ + 2 * H, D, generator=g).to(torch.bfloat16)
        qkv.copy_(rows)
        out.fill_(3.0)
        keep.copy_(_i32([len(k) for k in ks]))
        n_new.copy_(_i32(new))
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        lo = 0
        for b, n in enumerate(new):
            ks[b] = torch.cat([ks[b], rows[lo:lo + n, HQ:HQ + H].float()])
            vs[b] = torch.cat([vs[b], rows[lo:lo + n, HQ + H:].float()])
            for got, (window, sinks) in ((out, (0, 0)), (wout, (20, 2))):
                want, mag = ao.chunk_attention(rows[lo:lo + n, :HQ], ks[b], vs[b], window, sinks)
                err = (got[lo:lo + n].double().cpu() - want).abs()
                assert bool((err <= _tolerance(want, mag, len(ks[b]), torch.bfloat16, 6.0)).all()), (i, b, window)
            lo += n
        assert bool((out[lo:] == 3).all()) and status.item() == 0
    pages.check_status()


def test_a_cache_past_32_bits_of_elements(cuda_lib):
    """A pool of more than 2^32 bytes and 2^31 elements, the request's pages at its end."""
    P, page_len, H, D = 1 << 17, 16, 8, 128
    pool = torch.empty(1, P, 2, page_len, H, D, dtype=torch.bfloat16, device=DEV)  # 8.6 GB, 4.3e9 elements
    c = _setup(17, [33, 1], [500, 700], 16, 8)
    table = c["table"] + (P - c["pool"].shape[1])
    pool[0, P - c["pool"].shape[1]:] = c["pool"][1].to(DEV)
    plan = dict(page_table=table.to(DEV), kv_len=_i32(c["kv_len"]), q_indptr=_i32(c["indptr"]))
    _check(c, chunk_attention_paged(c["q"].to(DEV), pool, 0, **plan))
    slots = torch.tensor([P * page_len - 1, (P - 1) * page_len], device=DEV)
    rows = torch.randn(2, H, D, device=DEV).to(torch.bfloat16)
    append_paged_kv_slots(pool, 0, rows, rows + 1, slot_map=slots)
    assert torch.equal(pool[0, P - 1, 0, page_len - 1], rows[0]) and torch.equal(pool[0, P - 1, 1, 0], (rows + 1)[1])


def test_prompts_into_the_loop(cuda_lib):
    """Prompts enter a speculative loop in two chunks, then a tree step runs behind them: the pages, the cache rows and
    both attentions are those of one request at a time."""
    H, HQ, D, nodes = 2, 8, 128, 6
    g = torch.Generator().manual_seed(18)
    loop = SpeculativeLoopBatch(2, nodes, DEV, kv_layers=1, kv_heads=H, head_dim=D, page_len=16, pages_per_seq=12, init_len=0,
                                max_chunk_tokens=120)
    ks, vs = [torch.zeros(0, H, D)] * 2, [torch.zeros(0, H, D)] * 2
    for new in ([50, 17], [0, 63], [1, 1]):
        plan = loop.begin_chunk(_i32(new))
        T = sum(new)
        q, k, v = (torch.randn(T, h, D, generator=g).to(torch.bfloat16) for h in (HQ, H, H))
        append_paged_kv_slots(loop.pool, 0, k.to(DEV), v.to(DEV), slot_map=plan.slot_map, status=loop.status)
        out = chunk_attention_paged(q.to(DEV), loop.pool, 0, page_table=plan.page_table, kv_len=plan.kv_len,
                                    q_indptr=plan.q_indptr, status=loop.status)
        lo = 0
        for b, n in enumerate(new):
            ks[b], vs[b] = torch.cat([ks[b], k[lo:lo + n].float()]), torch.cat([vs[b], v[lo:lo + n].float()])
            want, mag = ao.chunk_attention(q[lo:lo + n], ks[b], vs[b])
            err = (out[lo:lo + n].double().cpu() - want).abs()
            assert bool((err <= _tolerance(want, mag, len(ks[b]), torch.bfloat16, 6.0)).all())
            lo += n
    assert loop.state.kv_len.tolist() == [51, 81] and loop.pages.kv_len.tolist() == [51, 81]
    # the tree step behind the prompts: a chain, so that its mask is the causal one and both attentions agree
    pos = loop.begin_step(nodes)
    assert loop.pages.kv_len.tolist() == [57, 87] and pos.positions[:nodes].tolist() == list(range(51, 57))
    from subspec_b200.attention import append_paged_kv
    q, k, v = (torch.randn(2, nodes, h, D, generator=g).to(torch.bfloat16).to(DEV) for h in (HQ, H, H))
    append_paged_kv(loop.pool, 0, k, v, page_table=loop.page_table, kv_len=loop.pages.kv_len)
    mask = torch.zeros(2, nodes, 96, dtype=torch.bool, device=DEV)
    for b, base in enumerate((51, 81)):
        for i in range(nodes):
            mask[b, i, :base + i + 1] = True
    tree = tree_attention_paged(q, loop.pool, 0, page_table=loop.page_table, kv_len=loop.pages.kv_len, mask=mask)
    flat = chunk_attention_paged(q.reshape(2 * nodes, HQ, D), loop.pool, 0, page_table=loop.page_table,
                                 kv_len=loop.pages.kv_len, q_indptr=_i32([0, nodes, 2 * nodes]))
    # each is within its own roundings of the same sum: weights and output rounded to bf16 on both sides
    assert float((tree.float() - flat.view_as(tree).float()).abs().max()) <= 4 * 2 ** -8 * float(tree.float().abs().max())
    assert loop.status.item() == 0
    loop.pages.check_status()


# ---------------------------------------------------------------- batches of many short chunks

def _dense(q, k, v, window=0, sinks=0):
    """`ao.chunk_attention` of finite rows with a dense mask (no loop over tokens)."""
    n, HQ, D = q.shape
    kv_len, G = k.shape[0], HQ // k.shape[1]
    qd, kd, vd = q.double().transpose(0, 1), *(x.double().repeat_interleave(G, 1).transpose(0, 1) for x in (k, v))
    p, j = torch.arange(kv_len - n, kv_len)[:, None], torch.arange(kv_len)[None, :]
    see = j <= p
    if window:
        see &= (j > p - window) | (j < sinks)
    w = torch.softmax((qd @ kd.transpose(1, 2) / D ** 0.5).masked_fill(~see, float("-inf")), -1)
    return (w @ vd).transpose(0, 1), (w @ vd.abs()).transpose(0, 1)


def _lengths(seed, count, lo, hi):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(lo, hi + 1, (count,), generator=g).tolist()


@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.float16)])
@pytest.mark.parametrize("new,cached,heads,kv_heads,window,sinks", [
    ([5] * 3, [0] * 3, 8, 1, 0, 0),
    ([20] * 3, [0] * 3, 4, 1, 0, 0),
    ([5, 5, 30, 5, 5, 5, 40], [0] * 7, 8, 1, 0, 0),
    ([20] * 64, [0] * 64, 32, 8, 0, 0),
    (_lengths(31, 64, 1, 300), [0] * 64, 32, 8, 0, 0),
    ([16] * 48, [100] * 48, 32, 8, 0, 0),
    ([6] * 256, _lengths(32, 256, 30, 200), 28, 4, 0, 0),
    (_lengths(33, 128, 8, 18), _lengths(34, 128, 0, 200), 28, 4, 0, 0),
    ([16] * 64, [300] * 64, 32, 8, 100, 0),
    (_lengths(35, 150, 3, 70), _lengths(36, 150, 0, 400), 8, 2, 60, 5),
    ([17] * 300, [0] * 300, 16, 8, 0, 0),
], ids=lambda x: None if isinstance(x, list) else str(x))
def test_many_short_chunks(cuda_lib, new, cached, heads, kv_heads, window, sinks, D, dtype):
    """Batches whose row tiles have up to 128 rows, the second block of a CTA none, one behind the other: every row
    is written (the output starts as NaN), nothing is reported, the values are the formula's."""
    c = _setup(37, new, cached, heads, kv_heads, D=D, dtype=dtype, layers=1, layer=0)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    for kw in (dict(), dict(max_q_len=max(new))):
        out = torch.full(c["q"].shape, float("nan"), dtype=dtype, device=DEV)
        got = _run(c, window, sinks, status, out=out, **kw).double().cpu()
        assert status.item() == 0
        for b, n in enumerate(new):
            lo = c["indptr"][b]
            want, mag = _dense(c["q"][lo:lo + n], c["ks"][b], c["vs"][b], window, sinks)
            err = (got[lo:lo + n] - want).abs()
            assert bool((err <= _tolerance(want, mag, c["kv_len"][b], dtype, 6.0)).all()), b


# ---------------------------------------------------------------- pages given back behind a window

def _give_back(pages, b, first, last):
    """Entries [first, last) of request b's list: -1 in the table, free in the mask."""
    for j in range(first, last):
        p = int(pages.page_table[b, j])
        pages.page_table[b, j] = -1
        pages.free_mask[p // 32] |= 1 << p % 32 if p % 32 < 31 else -2 ** 31  # (the words are signed)


@pytest.mark.parametrize("release", ["plan", "update", "cut"])
def test_requests_that_gave_pages_back_go_on_and_finish(cuda_lib, release):
    """Plan, give back the pages behind the window, plan more tokens (which get those pages), attend, finish: nothing
    is reported, no page is lost.  A page id outside the pool is reported as before."""
    H, HQ, D, page_len, P = 2, 4, 64, 16, 70
    g = torch.Generator().manual_seed(41)
    pages = DevicePagePool(2, P, page_len, 64, DEV, max_append=700)
    pool = torch.full((1, P, 2, page_len, H, D), float("nan"), dtype=torch.float16, device=DEV)
    ks, vs = [torch.zeros(0, H, D)] * 2, [torch.zeros(0, H, D)] * 2

    def step(new, window, sinks):
        plan = pages.plan_chunks(_i32(new))
        q, k, v = (torch.randn(sum(new), h, D, generator=g).to(torch.float16) for h in (HQ, H, H))
        append_paged_kv_slots(pool, 0, k.to(DEV), v.to(DEV), slot_map=plan.slot_map)
        status = torch.zeros(1, dtype=torch.int32, device=DEV)
        out = window_attention_paged(q.to(DEV), pool, 0, page_table=plan.page_table, kv_len=plan.kv_len,
                                     q_indptr=plan.q_indptr, window=window, sinks=sinks, status=status)
        assert status.item() == 0
        lo = 0
        for b, n in enumerate(new):
            ks[b], vs[b] = torch.cat([ks[b], k[lo:lo + n].float()]), torch.cat([vs[b], v[lo:lo + n].float()])
            want, mag = _dense(q[lo:lo + n], ks[b], vs[b], window, sinks)
            err = (out[lo:lo + n].double().cpu() - want).abs()
            assert bool((err <= _tolerance(want, mag, len(ks[b]), torch.float16, 6.0)).all())
            lo += n

    step([600, 40], 100, 5)                      # 38 and 3 pages
    assert pages.num_free_pages() == P - 41
    _give_back(pages, 0, 1, 31)                  # rows 16 .. 495; the next token's window begins at row 501
    assert pages.num_free_pages() == P - 11
    step([20, 500], 100, 5)                      # the second request takes pages that the first gave back
    assert pages.n_pages.tolist() == [39, 34] and set(pages.page_table[1, 3:34].tolist()) & set(range(1, 31))
    pages.check_status()
    if release == "cut":                         # back into the part that is gone, then on to nothing
        pages.plan_chunks(_i32([0, 0]), set_len=_i32([200, 10]))
        assert pages.n_pages.tolist() == [13, 1] and pages.num_free_pages() == P - 2
        pages.check_status()
    if release == "update":
        pages.update(set_len=_i32([0, 0]), mode="prefill")
    else:
        pages.plan_chunks(_i32([0, 0]), set_len=_i32([0, 0]))
    pages.check_status()
    assert pages.num_free_pages() == P and pages.n_pages.tolist() == [0, 0] and bool((pages.free_mask[:2] == -1).all())
    for finish in (lambda: pages.update(set_len=_i32([0, 0]), mode="prefill"),
                   lambda: pages.plan_chunks(_i32([0, 0]), set_len=_i32([0, 0]))):
        pages.plan_chunks(_i32([40, 0]))
        for bad in (P, -2):
            pages.page_table[0, 1] = bad
        finish()
        with pytest.raises(ValueError, match="page"):
            pages.check_status()


@pytest.mark.parametrize("D,dtype,per", [(128, torch.bfloat16, 2), (64, torch.float16, 4), (128, torch.float16, 6)])
def test_many_rows_done_over(cuda_lib, D, dtype, per):
    """Short chunks whose last token's V row holds an infinity in every dim: all rows in front of it are written twice, by
    the tile (0 * inf) and key by key.  The second writing is what stays, call after call."""
    B, heads, kv_heads = 200, 8, 2
    c = _setup(43, [per] * B, _lengths(44, B, 0, 60), heads, kv_heads, D=D, dtype=dtype)
    for b in range(B):
        j = c["kv_len"][b] - 1
        c["vs"][b][j] = float("inf")
        c["pool"][1, c["table"][b, j // 16], 1, j % 16] = float("inf")
    first = None
    for _ in range(20):
        got = _run(c, max_q_len=per)
        assert first is None or torch.equal(got, first)
        first = got
    got = first.view(B, per, heads, D).double().cpu()
    assert bool((got[:, -1] == float("inf")).all())
    for b in range(B):
        q = c["q"][b * per:(b + 1) * per - 1]
        want, mag = _dense(q, c["ks"][b][:-1], c["vs"][b][:-1])
        assert bool(((got[b, :-1] - want).abs() <= _tolerance(want, mag, c["kv_len"][b], dtype, 6.0)).all()), b


# ---------------------------------------------------------------- errors without a status word of the caller's

def test_errors_without_a_status_are_kept(cuda_lib):
    """Calls that leave `status` out report to the library's word of the device, eager and captured, which check_status
    reads and clears; calls that bring a word of their own leave it alone."""
    from subspec_b200.attention import check_status

    try:
        check_status()  # (what an earlier test may have left)
    except ValueError:
        pass
    for new in ([1, 1], [40, 40]):  # either kernel
        c = _setup(51, new, [60, 60], 4, 2)
        _run(c)
        check_status()
        good = c["table"].clone()
        c["table"][0, 1] = 10 ** 6
        own = torch.zeros(1, dtype=torch.int32, device=DEV)
        _run(c, status=own)
        check_status()
        assert own.item() == 8
        _check(c, _run(c), only=[1])
        with pytest.raises(ValueError, match="page"):
            check_status(DEV)
        check_status(torch.device(DEV, 0))
        c["table"] = good
        _run(c, window=30, max_q_len=new[0] - 1 or 0)
        if new[0] > 1:  # (max_q_len 0: nothing to do, nothing launched)
            with pytest.raises(ValueError, match="count"):
                check_status()
        check_status()
    pool = torch.zeros(1, 4, 2, 4, 2, 64, dtype=torch.bfloat16, device=DEV)
    k = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device=DEV)
    slots = torch.tensor([0, 16], device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        append_paged_kv_slots(pool, 0, k, k, slot_map=slots)
    check_status()
    graph.replay()
    with pytest.raises(ValueError, match="index"):
        check_status()
    slots.fill_(-1)
    graph.replay()
    check_status()
