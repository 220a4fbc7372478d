"""The serving step where its operators meet: steps that are refused, and maps longer than the step's rows."""
import random

import pytest

import test_gpu_serving_ops as ops
from test_gpu_serving_ops import DIM, PAGE, Pages, _ints, _stream

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------ the append of a planned step
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("nkv,layers,layer,rows,count", [(8, 1, 0, 1, 1), (1, 3, 2, 70, 70), (5, 2, 0, 333, 200), (8, 2, 1, 40, 0),
                                                         (8, 1, 0, 12, -3), (2, 1, 0, 9, 2**31 - 1), (8, 1, 0, 20000, 20000)])
def test_planned_append_writes_the_rows_that_were_given_out(qasr, cuda_device, nkv, layers, layer, rows, count, dtype):
    """Bit for bit, and nothing else: rows past the count, slots, positions and pages out of range."""
    import torch
    t = torch.bfloat16 if dtype == "bf16" else torch.float16
    slots, max_pages, pool_pages = 13, 40, 600
    rng = random.Random(rows)
    cells = rng.sample(range(slots * max_pages * PAGE), rows)  # distinct (slot, position)
    slot, pos = [c // (max_pages * PAGE) for c in cells], [c % (max_pages * PAGE) for c in cells]
    for i, (s, p) in enumerate([(-1, 0), (slots, 0), (0, -1), (0, max_pages * PAGE), (2**31 - 1, 2**31 - 1)]):
        if rows > 100:
            slot[7 * i], pos[7 * i] = s, p
    page = torch.randperm(pool_pages, device="cuda")[:slots * max_pages].to(torch.int32).view(slots, max_pages)
    page[3, 5], page[4, 0], page[0, 1] = -1, pool_pages, 2**31 - 1
    k, v = (torch.randn((rows, nkv * DIM), device="cuda").to(t) for _ in range(2))
    pool = torch.full((pool_pages, layers, 2, nkv, PAGE, DIM), 3.0, dtype=t, device="cuda")
    want = pool.clone()
    m = max(0, min(count, rows))
    s, p = (torch.tensor(x[:m], dtype=torch.int64, device="cuda") for x in (slot, pos))
    ok = (s >= 0) & (s < slots) & (p >= 0) & (p < max_pages * PAGE)
    s, p, kk, vv = s[ok], p[ok], k[:m][ok], v[:m][ok]
    pg = page[s, p // PAGE].long()
    ok = (pg >= 0) & (pg < pool_pages)
    pg, p, kk, vv = pg[ok], p[ok], kk[ok], vv[ok]
    d = torch.arange(DIM, device="cuda")
    col = (((d >> 3)[None, :] ^ (p & 7)[:, None]) << 3) | (d & 7)[None, :]
    for h in range(nkv):
        for part, x in enumerate((kk, vv)):
            want[pg[:, None], layer, part, h, (p % PAGE)[:, None], col] = x[:, h * DIM:(h + 1) * DIM]
    d_slot, d_pos, d_count = _ints(slot, torch), _ints(pos, torch), _ints([count], torch)
    qasr.kernel_kv_append_planned(0, _stream(torch), k.data_ptr(), v.data_ptr(), pool.data_ptr(), pool_pages, page.data_ptr(),
                                  slots, max_pages, layers, nkv, layer, d_slot.data_ptr(), d_pos.data_ptr(), rows,
                                  d_count.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(pool, want)


@pytest.mark.parametrize("rows_cap", [3, 8, 60000])  # exact maps, longer ones, maps that a second kernel writes
def test_a_captured_step_that_runs_out_of_pages_leaves_the_cache_alone(qasr, cuda_device, rows_cap):
    """Plan, append and attention in one graph, replayed until the free stack is empty: the refused step writes nothing, in
    spite of the maps that still hold the step before, and the steps before it only their own rows."""
    import torch
    n, slots, max_pages, pool_pages, nkv, nq = 3, 5, 4, 4, 8, 16
    p = Pages(torch, slots, max_pages, pool_pages, seed=3)
    slot, held = [4, 1, 2], [62, 20, 64]
    ops._check_plan(p, p.plan(qasr, slot, [0] * n, held), slot, [0] * n, held)
    d_slot, d_len, cu, status = _ints(slot, torch), _ints(held, torch), _ints([0] * (n + 1), torch), _ints([-9, -9], torch)
    # before the first step the maps are whatever the memory held
    maps = [torch.randint(-2**31, 2**31 - 1, (rows_cap,), dtype=torch.int32, device="cuda") for _ in range(2)]
    pool = torch.randn((pool_pages, 1, 2, nkv, PAGE, DIM), device="cuda").to(torch.float16)
    k, v = (torch.randn((rows_cap, nkv * DIM), device="cuda").to(torch.float16) for _ in range(2))
    q = torch.randn((rows_cap, nq * DIM), device="cuda").to(torch.float16)
    out = torch.full_like(q, 77)
    ws_bytes = qasr.kernel_attention_chunk_workspace(0)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device="cuda")

    def step():
        st = _stream(torch)
        qasr.kernel_kv_plan(0, st, d_slot.data_ptr(), d_len.data_ptr(), None, n, slots, p.d_table.data_ptr(), max_pages,
                            p.d_free.data_ptr(), pool_pages, p.d_count.data_ptr(), d_len.data_ptr(), p.d_count.data_ptr(),
                            cu.data_ptr(), maps[0].data_ptr(), maps[1].data_ptr(), rows_cap, status.data_ptr())
        qasr.kernel_kv_append_planned(0, st, k.data_ptr(), v.data_ptr(), pool.data_ptr(), pool_pages, p.d_table.data_ptr(),
                                      slots, max_pages, 1, nkv, 0, maps[0].data_ptr(), maps[1].data_ptr(), rows_cap,
                                      cu.data_ptr() + 4 * n)
        qasr.kernel_attention_chunk(0, st, qasr.TYPE_F16, q.data_ptr(), nq * DIM, out.data_ptr(), nq * DIM, rows_cap,
                                    pool.data_ptr(), pool_pages, p.d_table.data_ptr(), slots, max_pages, 1, nq, nkv, 0,
                                    d_slot.data_ptr(), cu.data_ptr(), d_len.data_ptr(), n, ws.data_ptr(), ws_bytes)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    # one page is left, taken by the third request's first step; the first request wants another one in its third
    for i, refused in enumerate([False, False, True, True]):
        for x in (k, v, q):
            x.copy_(torch.randn_like(x))
        out.fill_(77)
        before = pool.clone()
        graph.replay()
        torch.cuda.synchronize()
        if refused:
            assert status.tolist() == [3, -1] and d_len.tolist() == held and cu.tolist() == [0] * (n + 1)
            assert torch.equal(pool, before) and (out == 77).all()
            continue
        p.expect(slot, held, [1] * n)
        assert status.tolist() == [0, 0] and p.d_table.tolist() == p.table
        for r, (s, pos) in enumerate(zip(slot, held)):
            d = torch.arange(DIM, device="cuda")
            col = (((d >> 3) ^ (pos & 7)) << 3) | (d & 7)
            for part, x in enumerate((k, v)):
                before[p.table[s][pos // PAGE], 0, part, :, pos % PAGE, col] = x[r].view(nkv, DIM)
        held = [h + 1 for h in held]
        assert torch.equal(pool, before) and d_len.tolist() == held
        assert out[:n].isfinite().all() and (out[:n] != 77).any() and (out[n:] == 77).all()


# ------------------------------------------------------------------------------------ waits that gave up
@pytest.mark.parametrize("cta", [0, 77, -1])
def test_a_wait_that_gave_up_is_told_however_many_calls_follow(qasr, cuda_device, cta):
    """The mark that a call leaves in its CTA's line of the workspace (written here from the host, four words from byte
    32 on) outlives the calls after it, eager and captured, until the check has told it once."""
    import torch
    c = ops.Chunks(torch, [(700, 90), (1200, 1), (0, 300)], seed=30)
    ws = c.workspace(qasr)
    c.run(qasr, ws=ws)
    qasr.kernel_attention_chunk_check(0, _stream(torch), ws[0].data_ptr())
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    mark = torch.tensor([(0x6c6f7374 * (2 * i + 1) + 0x9e3779b9) % 2**32 for i in range(4)], dtype=torch.uint32, device="cuda")
    ws[0].view(torch.uint32)[:16 * sms].view(sms, 16)[cta, 8:12] = mark
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        c.run(qasr, ws=ws)
    for _ in range(3):
        c.run(qasr, ws=ws)
        graph.replay()
    with pytest.raises(qasr.DecoderError) as e:
        qasr.kernel_attention_chunk_check(0, _stream(torch), ws[0].data_ptr())
    assert e.value.status == 5
    qasr.kernel_attention_chunk_check(0, _stream(torch), ws[0].data_ptr())
    c.run(qasr, ws=ws)
    qasr.kernel_attention_chunk_check(0, _stream(torch), ws[0].data_ptr())
    c.check(c.out)


# ------------------------------------------------------------------------------------ scores that are not numbers
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("at", [0, 5, 6, 7, 14, 15, 62, 63, 64 + 6, 128 + 31])
def test_a_key_that_is_not_a_number_among_keys_of_minus_infinity(qasr, cuda_device, at, dtype):
    """One NaN key, every other key of the first 1024 positions so low that its score is -inf: the running maximum passes
    over both.  Every row that sees the NaN is NaN, in a prompt, a short chunk, a whole decode row and one whose keys
    are cut over CTAs, the other parts of which are finite; rows before it are NaN too, softmax of nothing but -inf."""
    import torch
    c = ops.Chunks(torch, [(0, 200), (160, 20), (250, 1), (9000, 1)], seed=31, dtype=dtype)
    c.q.abs_().add_(0.01)
    for kv in c.kv:
        kv[0, :, :1024] = -float("inf")
        kv[0, :, at] = float("nan")
    c.store()
    out = c.run(qasr)
    torch.cuda.synchronize()
    assert out[:222, :2048].isnan().all()


# ------------------------------------------------------------------------------------ scales
@pytest.mark.parametrize("scale,size", [(1e-33, 1e16), (-1e-33, 1e16), (1e-37, 1e18), (0.0, 1e18), (0.0, 1.0), (1e-30, 1e15),
                                        (1e20, 1e-10), (1.5e38, 0.0)])
def test_chunk_attention_takes_scales_of_any_size(qasr, cuda_device, scale, size):
    """Tiny scales under huge scores, 0 among them, and the other way round (bf16 has the range for it)."""
    import torch
    c = ops.Chunks(torch, [(0, 100), (300, 1), (64, 64)], seed=32, dtype="bf16")
    c.q *= size
    for kv in c.kv:
        kv[0] *= size
    c.store()
    out = c.run(qasr, scale=scale)
    torch.cuda.synchronize()
    c.check(out, scale=scale)


# ------------------------------------------------------------------------------------ values that are not finite
def _expect_not_finite(c, out, torch):
    """NaN, infinities and finite outputs where the formula in 64 bits has them: a probability above 0 times an infinite value
    is infinite, times NaN is NaN, and what a row does not see does not count."""
    first, G = 0, c.nq // c.nkv
    for i, (a, b) in enumerate(c.lens):
        v = c.kv[i][1].float()  # [nkv, positions, dims]
        seen = [flag.cumsum(1)[:, a:a + b] > 0 for flag in (v.isnan(), v == torch.inf, v == -torch.inf)]
        nan, plus, minus = (x.permute(1, 0, 2).repeat_interleave(G, 1) for x in seen)  # [rows, nq, dims]
        nan = nan | (plus & minus)
        got = out[first:first + b, :c.nq * DIM].view(b, c.nq, DIM)
        assert torch.equal(got.isnan(), nan), i
        assert torch.equal(got == torch.inf, plus & ~nan) and torch.equal(got == -torch.inf, minus & ~nan), i
        first += b


def _zeroed(c, torch):
    """0 for each value that is not finite."""
    for x in c.kv:
        x[1] = torch.where(x[1].isfinite(), x[1], torch.zeros_like(x[1]))


LENS = [(0, 300), (90, 20), (500, 1), (3000, 1), (2000, 130), (0, 64)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("value", ["nan", "inf", "-inf", "both", "mixed"])
@pytest.mark.parametrize("where", ["first", "few", "late", "one dim", "all"])
def test_chunk_attention_of_values_that_are_not_finite(qasr, cuda_device, where, value, dtype):
    """Prompts, short chunks, whole and cut decode rows, with values that are not finite at the first position, at
    some, at late ones only (masked for earlier rows of the same block), in one dim, everywhere.  Scores spread so far
    that f16 probabilities vanish beside the largest; an infinite value still counts there."""
    import torch
    c = ops.Chunks(torch, LENS, seed=33, dtype=dtype, spread=2.5)
    rng = random.Random(7)
    kinds = {"nan": ["nan"], "inf": ["inf"], "-inf": ["-inf"], "both": ["inf", "-inf"], "mixed": ["nan", "inf", "-inf"]}[value]
    for kv in c.kv:
        n = kv.shape[2]
        at = {"first": [0], "few": [rng.randrange(n) for _ in range(5)], "late": [n - 1 - rng.randrange(min(n, 40)) for _ in range(3)],
              "one dim": [rng.randrange(n) for _ in range(3)], "all": range(n)}[where]
        for t in at:
            dims = slice(0, DIM) if where != "one dim" else rng.randrange(DIM)
            kv[1, :, t, dims] = float(rng.choice(kinds))
    c.store()
    out = c.run(qasr)
    torch.cuda.synchronize()
    _expect_not_finite(c, out, torch)
    # what stays finite, against the formula
    _zeroed(c, torch)
    got = out.clone()
    d = ops.Chunks(torch, LENS, seed=33, dtype=dtype, spread=2.5)
    d.kv = c.kv
    d.store()
    clean = d.run(qasr)
    torch.cuda.synchronize()
    d.check(torch.where(got.isfinite(), got, clean))


@pytest.mark.parametrize("what,times", [("nan", 30), ("inf", 30), ("one dim", 30), ("late", 200), ("key", 3)])
def test_one_value_that_is_not_finite_does_not_hold_up_the_call(qasr, cuda_device, what, times):
    """2048 rows, all of which see it: within 30 times the clean call (about 7 here, 460 when every such row was computed
    again); when it is masked for most rows of the last block, those are, within 200 times (about 95 here)."""
    import torch
    c = ops.Chunks(torch, [(0, 2048)], seed=34)
    ws = c.workspace(qasr)

    def fastest():
        best = 1e9
        for _ in range(5):
            a, b = torch.cuda.Event(True), torch.cuda.Event(True)
            a.record()
            c.run(qasr, ws=ws)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    clean = fastest()
    x = c.kv[0]
    if what == "key":
        x[0, :, 0] = float("nan")
    elif what == "one dim":
        x[1, :, 0, 5] = float("nan")
    else:
        x[1, :, 2000 if what == "late" else 0] = float("inf" if what == "inf" else "nan")
    c.store()
    broken = fastest()
    assert broken < times * clean


# ------------------------------------------------------------------------------------ plans
@pytest.mark.parametrize("rows", [32767, 32768, 32769, 49152, 49153])
@pytest.mark.parametrize("spare", [0, 1])
def test_kv_plan_where_the_maps_go_to_a_second_kernel(qasr, cuda_device, rows, spare):
    """The last rows that the planning kernel writes itself and the first that it leaves to the other one, by the room in
    the maps, which is what is known on the host."""
    import torch
    rng = random.Random(rows)
    new = [rng.randint(0, 1000) for _ in range(60)]
    new.append(rows - sum(new))
    assert new[-1] >= 0
    n, max_pages = len(new), -(-max(new) // PAGE)
    p = Pages(torch, n, max_pages, n * max_pages, seed=4)
    slot = rng.sample(range(n), n)
    ops._check_plan(p, p.plan(qasr, slot, [0] * n, new, rows_cap=rows + spare), slot, [0] * n, new)


@pytest.mark.parametrize("slot,held,count,want", [
    ([0, 5], [0, 0], 8, [1, 1]), ([-1, 0], [0, 0], 8, [1, 0]), ([1, 0, 1], [0, 0, 0], 8, [1, 2]), ([1, 0], [257, 0], 8, [1, 0]),
    ([1, 0], [0, -1], 8, [1, 1]), ([1, 0], [64, 64], -1, [1, -3]), ([1, 0], [64, 64], 21, [1, -3]), ([1, 0], [64, 64], 19, [3, -1]),
], ids=lambda v: str(v)[:24])
def test_kv_release_refuses_on_the_device_and_changes_nothing(qasr, cuda_device, slot, held, count, want):
    import torch
    p = Pages(torch, 5, 4, 20)
    p.d_count.fill_(count)
    s, h, st = _ints(slot, torch), _ints(held, torch), _ints([-9, -9], torch)
    qasr.kernel_kv_release(0, _stream(torch), s.data_ptr(), h.data_ptr(), len(slot), 5, p.d_table.data_ptr(), 4,
                           p.d_free.data_ptr(), 20, p.d_count.data_ptr(), h.data_ptr(), p.d_count.data_ptr(), st.data_ptr())
    torch.cuda.synchronize()
    assert st.tolist() == want and h.tolist() == held and p.d_count.item() == count
    assert p.d_free.tolist() == p.free and p.d_table.tolist() == p.table


# ------------------------------------------------------------------------------------ outputs written anew
def test_chunk_attention_on_two_streams_writes_every_row_each_time(qasr, cuda_device):
    """Two calls at once, each output wiped before each run and compared after it."""
    import torch
    c = ops.Chunks(torch, [(700, 90), (1200, 1), (0, 300)] * 3, seed=14)
    d = ops.Chunks(torch, [(2500, 1)] * 20, seed=15, dtype="bf16")
    a, b = c.run(qasr).clone(), d.run(qasr).clone()
    wc, wd = c.workspace(qasr), d.workspace(qasr)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        c.out.fill_(77)
        d.out.fill_(77)
        torch.cuda.synchronize()
        c.run(qasr, ws=wc, stream=s1.cuda_stream)
        d.run(qasr, ws=wd, stream=s2.cuda_stream)
        torch.cuda.synchronize()
        assert torch.equal(a, c.out) and torch.equal(b, d.out)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("which", [0, 1])
def test_chunk_attention_writes_the_rows_before_a_broken_position(qasr, cuda_device, which, value):
    import torch
    c = ops.Chunks(torch, [(90, 200), (0, 40), (300, 1)], seed=10)
    kv = [x.clone() for x in c.kv]
    c.kv[0][which, :, 90 + 150] = value
    c.kv[1][which, :, 39] = value
    c.store()
    out = c.run(qasr)  # into an output that no run has written
    torch.cuda.synchronize()
    c.kv = kv
    c.check(out, skip=set(range(150, 200)) | {239})


def test_calls_for_another_device_leave_the_current_one_alone(qasr, cuda_device):
    import torch
    if torch.cuda.device_count() < 2:
        pytest.skip("one device")
    w = ops.W4(qasr, torch, 64, 64, 64, False, "f16", 1)
    c = ops.Chunks(torch, [(0, 4)])
    stream = torch.cuda.current_stream(0).cuda_stream
    torch.cuda.synchronize()
    with torch.cuda.device(1):
        qasr.kernel_gemv_w4(0, stream, qasr.TYPE_F16, w.packed.data_ptr(), False, 64, 64, 64, w.x.data_ptr(), 64, 1,
                            w.out.data_ptr(), 64)
        c.run(qasr, stream=stream)
        assert torch.cuda.current_device() == 1
    torch.cuda.synchronize()
    w.check(w.out)
    c.check(c.out)


# ------------------------------------------------------------------------------------ a step of all operators, bf16, room to spare
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_a_captured_serving_step_with_room_for_more_rows(qasr, cuda_device, dtype):
    """Plan, 4-bit q|k|v product, planned append, attention, 4-bit output product in one graph with room for 64 rows,
    replayed with chunks, single tokens, an idle request and a step that is refused in between."""
    import torch
    t = torch.bfloat16 if dtype == "bf16" else torch.float16
    hs, nq, nkv, max_pages, slots, pool_pages, cap, n = 512, 16, 8, 4, 6, 14, 64, 3
    p = Pages(torch, slots, max_pages, pool_pages, seed=8)
    pool = torch.full((pool_pages, 1, 2, nkv, PAGE, DIM), float("nan"), dtype=t, device="cuda")
    qkv = ops.W4(qasr, torch, (nq + 2 * nkv) * DIM, hs, 64, True, dtype, cap, seed=1)
    o = ops.W4(qasr, torch, hs, nq * DIM, 128, False, dtype, cap, seed=2)
    qkv.scale.mul_(0.3)
    qasr.kernel_pack_w4(0, _stream(torch), qkv.codes.data_ptr(), qkv.scale.data_ptr(), qkv.zero.data_ptr(), qkv.n_out, hs, 64,
                        qkv.packed.data_ptr())
    ws_bytes = qasr.kernel_attention_chunk_workspace(0)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device="cuda")
    slot, held = [4, 0, 3], [0, 0, 0]
    d_slot, d_len, d_new = _ints(slot, torch), _ints(held, torch), _ints([0] * n, torch)
    cu, status = _ints([0] * (n + 1), torch), _ints([0, 0], torch)
    maps = [_ints([2**31 - 1] * cap, torch) for _ in range(2)]
    k, v = (torch.empty((cap, nkv * DIM), dtype=t, device="cuda") for _ in range(2))
    att = torch.empty((cap + 1, nq * DIM), dtype=t, device="cuda")
    y = qkv.out
    o.x = att

    def step():
        st = _stream(torch)
        qasr.kernel_kv_plan(0, st, d_slot.data_ptr(), d_len.data_ptr(), d_new.data_ptr(), n, slots, p.d_table.data_ptr(), max_pages,
                            p.d_free.data_ptr(), pool_pages, p.d_count.data_ptr(), d_len.data_ptr(), p.d_count.data_ptr(),
                            cu.data_ptr(), maps[0].data_ptr(), maps[1].data_ptr(), cap, status.data_ptr())
        qkv.run(qasr)
        k.copy_(y[:cap, nq * DIM:(nq + nkv) * DIM])
        v.copy_(y[:cap, (nq + nkv) * DIM:])
        qasr.kernel_kv_append_planned(0, st, k.data_ptr(), v.data_ptr(), pool.data_ptr(), pool_pages, p.d_table.data_ptr(), slots,
                                      max_pages, 1, nkv, 0, maps[0].data_ptr(), maps[1].data_ptr(), cap, cu.data_ptr() + 4 * n)
        qasr.kernel_attention_chunk(0, st, qasr.TYPE_BF16 if dtype == "bf16" else qasr.TYPE_F16, y.data_ptr(), y.shape[1],
                                    att.data_ptr(), nq * DIM, cap, pool.data_ptr(), pool_pages, p.d_table.data_ptr(), slots,
                                    max_pages, 1, nq, nkv, 0, d_slot.data_ptr(), cu.data_ptr(), d_len.data_ptr(), n, ws.data_ptr(),
                                    ws_bytes)
        o.run(qasr, accumulate=True)

    step()  # a step of no rows: also the first call of each, ahead of the capture
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    cache = {s: torch.empty((2, nkv, 0, DIM), dtype=t, device="cuda") for s in slot}
    for new, refused in [([30, 21, 13], 0), ([1, 1, 1], 0), ([40, 40, 1], 1), ([20, 0, 40], 0), ([1, 300, 1], 1), ([1, 1, 1], 0)]:
        d_new.copy_(_ints(new, torch))
        qkv.x.copy_(torch.randn_like(qkv.x))
        att.fill_(77)
        o.out[:cap] = torch.randn((cap, hs), device="cuda").to(t)
        resid, before = o.out[:cap].clone(), pool.clone()
        graph.replay()
        qasr.kernel_attention_chunk_check(0, _stream(torch), ws.data_ptr())
        qasr.kernel_gemv_w4_check(0, _stream(torch))
        torch.cuda.synchronize()
        qkv.check(y)
        if refused:
            assert status.tolist()[0] == 3 and d_len.tolist() == held
            assert torch.equal(pool.view(torch.int16), before.view(torch.int16)) and (att == 77).all()
            continue
        rows = sum(new)
        p.expect(slot, held, new)
        assert status.tolist() == [0, 0] and p.d_table.tolist() == p.table
        c = ops.Chunks.__new__(ops.Chunks)
        c.torch, c.t, c.nq, c.nkv, c.rows, c.lens = torch, t, nq, nkv, rows, list(zip(held, new))
        c.q, c.kv, first = y[:, :nq * DIM], [], 0
        for i, s in enumerate(slot):
            add = torch.stack([k[first:first + new[i]], v[first:first + new[i]]]).view(2, new[i], nkv, DIM).transpose(1, 2)
            cache[s] = torch.cat([cache[s], add], 2)
            c.kv.append(cache[s])
            first += new[i]
        c.check(att)
        held = [a + b for a, b in zip(held, new)]
        assert d_len.tolist() == held
        o.x = att[:cap]
        o.check(o.out, before=resid)
        o.x = att
