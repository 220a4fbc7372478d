"""The serving step's operators on the B200 against plain implementations: page and row maps against a
Python allocator (exact), chunk attention and 4-bit products against 64-bit torch, each at the sizes, masks and
layouts where they can go wrong, then all of them run together.

Tolerances are bounds of the arithmetic, written where they are used; u is half a step of the output type."""
import random

import pytest

pytestmark = pytest.mark.gpu

PAGE, DIM = 64, 128


def _ints(values, torch):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _stream(torch):
    return torch.cuda.current_stream().cuda_stream


# ------------------------------------------------------------------------------------ page and row maps
class Pages:
    """The allocator's device state and its plain double."""

    def __init__(self, torch, slots, max_pages, pool_pages, seed=0, spare_rows=8):
        self.torch, self.slots, self.max_pages, self.pool_pages = torch, slots, max_pages, pool_pages
        order = list(range(pool_pages))
        random.Random(seed).shuffle(order)
        self.free, self.table = order, [[-1] * max_pages for _ in range(slots)]
        self.d_table = _ints(self.table, torch)
        self.d_free = _ints(order, torch)
        self.d_count = _ints([pool_pages], torch)

    def plan(self, qasr, slot, held, new, rows_cap=None, alias=True, pass_new=True):
        t, n = self.torch, len(slot)
        total = sum(new)
        cap = total if rows_cap is None else rows_cap
        s, h, a = _ints(slot, t), _ints(held, t), _ints(new, t)
        out = h if alias else t.full_like(h, -7)
        count_out = self.d_count if alias else t.full_like(self.d_count, -7)
        cu = t.full((n + 2,), -9, dtype=t.int32, device="cuda")
        maps = [t.full((cap + 8,), -9, dtype=t.int32, device="cuda") for _ in range(2)]
        status = t.full((2,), -9, dtype=t.int32, device="cuda")
        qasr.kernel_kv_plan(0, _stream(t), s.data_ptr(), h.data_ptr(), a.data_ptr() if pass_new else None, n, self.slots,
                            self.d_table.data_ptr(), self.max_pages, self.d_free.data_ptr(), self.pool_pages,
                            self.d_count.data_ptr(), out.data_ptr(), count_out.data_ptr(), cu.data_ptr(),
                            maps[0].data_ptr(), maps[1].data_ptr(), cap, status.data_ptr())
        t.cuda.synchronize()
        got = dict(out=out.tolist(), count=count_out.tolist()[0], cu=cu.tolist(), slot=maps[0].tolist(),
                   pos=maps[1].tolist(), status=status.tolist(), table=self.d_table.tolist())
        self.d_count.copy_(count_out)
        return got

    def expect(self, slot, held, new):
        """The same step on the host's double; returns (cu, row_slot, row_pos)."""
        cu, rs, rp = [0], [], []
        for s, h, a in zip(slot, held, new):
            for j in range(-(-h // PAGE), -(-(h + a) // PAGE)):
                self.table[s][j] = self.free.pop()
            rs += [s] * a
            rp += range(h, h + a)
            cu.append(len(rs))
        return cu, rs, rp


def _check_plan(p, got, slot, held, new):
    cu, rs, rp = p.expect(slot, held, new)
    assert got["status"] == [0, 0]
    assert got["cu"] == cu + [-9]
    assert got["slot"][:len(rs)] == rs and set(got["slot"][len(rs):]) == {-9}
    assert got["pos"][:len(rp)] == rp and set(got["pos"][len(rp):]) == {-9}
    assert got["out"] == [h + a for h, a in zip(held, new)]
    assert got["count"] == len(p.free)
    assert got["table"] == p.table


@pytest.mark.parametrize("n,slots,hi,alias", [
    (1, 1, 1, True), (1, 3, 64, False), (2, 2, 65, True), (33, 40, 200, False), (256, 256, 30, True),
    (257, 300, 1, True), (700, 700, 150, False), (1025, 2000, 9, True), (8192, 8192, 3, True), (5, 65536, 5000, False),
])
def test_kv_plan_matches_a_plain_allocator(qasr, cuda_device, n, slots, hi, alias):
    """Three steps in a row: lengths of zero and more, page borders met from below, on and above them."""
    import torch
    rng = random.Random(n * 31 + hi)
    max_pages = -(-3 * (hi + PAGE) // PAGE) + 1
    p = Pages(torch, slots, max_pages, n * max_pages + 5, seed=n)
    slot = rng.sample(range(slots), n)
    held = [0] * n
    for step in range(3):
        new = [rng.choice([0, 1, hi, rng.randint(0, hi), min(hi, -h % PAGE), min(hi, -h % PAGE + 1)]) for h in held]
        got = p.plan(qasr, slot, held, new, alias=alias, rows_cap=sum(new) + (step * 5))
        _check_plan(p, got, slot, held, new)
        held = got["out"]


@pytest.mark.parametrize("shift", [0, 1])
def test_kv_plan_long_row_maps(qasr, cuda_device, shift):
    """More rows than the planning cluster writes itself, runs of empty requests among them, maps on and off 16-byte
    boundaries, and more room than rows."""
    import torch
    rng = random.Random(shift)
    n, max_pages = 400, 40
    new = [rng.choice([0, 0, 1, 3, 64, 2000, rng.randint(0, 300)]) for _ in range(n)]
    new[:5], new[-6:] = [0] * 5, [0] * 6
    held = [rng.randint(0, 500) for _ in range(n)]
    assert sum(new) > 40000
    p = Pages(torch, n, max_pages, n * max_pages, seed=2)
    slot = rng.sample(range(n), n)
    first = p.plan(qasr, slot, [0] * n, held)
    _check_plan(p, first, slot, [0] * n, held)
    cu, rs, rp = p.expect(slot, held, new)
    s, h, a = _ints(slot, torch), _ints(held, torch), _ints(new, torch)
    maps = [torch.full((len(rs) + 100,), -9, dtype=torch.int32, device="cuda") for _ in range(2)]
    d_cu, st = _ints([0] * (n + 1), torch), _ints([-9, -9], torch)
    qasr.kernel_kv_plan(0, _stream(torch), s.data_ptr(), h.data_ptr(), a.data_ptr(), n, n, p.d_table.data_ptr(), max_pages,
                        p.d_free.data_ptr(), p.pool_pages, p.d_count.data_ptr(), h.data_ptr(), p.d_count.data_ptr(),
                        d_cu.data_ptr(), maps[0].data_ptr() + 4 * shift, maps[1].data_ptr() + 4 * shift, len(rs) + 90,
                        st.data_ptr())
    torch.cuda.synchronize()
    assert st.tolist() == [0, 0] and d_cu.tolist() == cu and p.d_count.item() == len(p.free)
    for got, want in zip(maps, (rs, rp)):
        got = got.tolist()
        assert got[shift:shift + len(want)] == want and set(got[shift + len(want):] + got[:shift]) == {-9}
    assert p.d_table.tolist() == p.table and h.tolist() == [x + y for x, y in zip(held, new)]


def test_kv_plan_without_new_lengths_adds_one_each(qasr, cuda_device):
    import torch
    p = Pages(torch, 9, 4, 30)
    slot, held = [8, 0, 3], [0, 0, 0]
    for new in ([63, 64, 127], [1, 1, 1], [1, 1, 1]):
        got = p.plan(qasr, slot, held, new, pass_new=new[0] != 1)
        _check_plan(p, got, slot, held, new)
        held = got["out"]


@pytest.mark.parametrize("alias", [True, False])
@pytest.mark.parametrize("slot,held,new,rows_cap,count,want", [
    ([0, 5, 1], [0, 0, 0], [1, 1, 1], 99, None, [1, 1]),             # slot past the table
    ([0, -1, 1], [0, 0, 0], [1, 1, 1], 99, None, [1, 1]),
    ([2, 1, 3, 1, 2], [0] * 5, [1] * 5, 99, None, [1, 3]),           # listed twice: the second listing
    ([0, 1, 2], [0, 257, 0], [1, 0, 1], 99, None, [1, 1]),           # holds more than its table has
    ([0, 1, 2], [0, 0, -1], [1, 1, 1], 99, None, [1, 2]),
    ([0, 1, 2], [0, 0, 0], [1, 1, -1], 99, None, [1, 2]),
    ([0, 1, 2], [0, 0, 0], [1, 1, 1], 99, -1, [1, -3]),              # a broken stack counter
    ([0, 1, 2], [0, 0, 0], [1, 1, 1], 99, 21, [1, -3]),
    ([0, 1, 2], [0, 200, 0], [1, 57, 1], 999, None, [3, 1]),         # past its table
    ([0, 1, 2], [0, 0, 0], [2**31 - 1, 1, 1], 99, None, [3, 0]),
    ([0, 1, 2], [0, 0, 0], [64, 64, 65], 999, 3, [3, -1]),           # the stack is one page short
    ([0, 1, 2], [0, 0, 0], [5, 6, 7], 17, None, [3, -2]),            # one row too many
    ([0, 1, 7], [0, 200, 0], [1, 57, 1], 99, None, [1, 2]),          # an invalid request before one that is full
], ids=lambda v: str(v)[:24])
def test_kv_plan_refuses_on_the_device_and_changes_nothing(qasr, cuda_device, slot, held, new, rows_cap, count, want, alias):
    import torch
    p = Pages(torch, 5, 4, 20)
    if count is not None:
        p.d_count.fill_(count)
    before = p.d_count.item()
    got = p.plan(qasr, slot, held, new, rows_cap=rows_cap, alias=alias)
    assert got["status"] == want
    assert got["cu"] == [0] * (len(slot) + 1) + [-9]
    assert got["out"] == held and got["count"] == before
    assert set(got["slot"]) == {-9} and set(got["pos"]) == {-9}
    assert got["table"] == p.table and p.d_free.tolist() == p.free


@pytest.mark.parametrize("n,slots", [(1, 1), (40, 64), (600, 640)])
def test_kv_release_gives_the_pages_back(qasr, cuda_device, n, slots):
    import torch
    rng = random.Random(n)
    p = Pages(torch, slots, 6, 6 * n + 2, seed=3)
    slot = rng.sample(range(slots), n)
    new = [rng.choice([0, 1, 64, 65, 6 * 64, rng.randint(0, 384)]) for _ in range(n)]
    got = p.plan(qasr, slot, [0] * n, new)
    _check_plan(p, got, slot, [0] * n, new)
    left = sorted(rng.sample(range(n), (n + 1) // 2))
    s, h = _ints([slot[i] for i in left], torch), _ints([new[i] for i in left], torch)
    status = _ints([-9, -9], torch)
    qasr.kernel_kv_release(0, _stream(torch), s.data_ptr(), h.data_ptr(), len(left), slots, p.d_table.data_ptr(), 6,
                           p.d_free.data_ptr(), p.pool_pages, p.d_count.data_ptr(), h.data_ptr(), p.d_count.data_ptr(),
                           status.data_ptr())
    torch.cuda.synchronize()
    for i in left:
        p.free += p.table[slot[i]][:-(-new[i] // PAGE)]
    assert status.tolist() == [0, 0] and h.tolist() == [0] * len(left)
    assert p.d_count.item() == len(p.free) and p.d_free[:len(p.free)].tolist() == p.free
    assert p.d_table.tolist() == p.table
    held = [p_ for i in range(n) if i not in left for p_ in p.table[slot[i]][:-(-new[i] // PAGE)]]
    assert sorted(held + p.free) == list(range(p.pool_pages))  # every page in one place


def test_kv_release_refuses_a_stack_that_would_overflow(qasr, cuda_device):
    import torch
    p = Pages(torch, 2, 4, 8)
    s, h, st = _ints([1, 0], torch), _ints([65, 0], torch), _ints([-9, -9], torch)
    free = p.d_free.clone()
    qasr.kernel_kv_release(0, _stream(torch), s.data_ptr(), h.data_ptr(), 2, 2, p.d_table.data_ptr(), 4,
                           p.d_free.data_ptr(), 8, p.d_count.data_ptr(), h.data_ptr(), p.d_count.data_ptr(), st.data_ptr())
    torch.cuda.synchronize()
    assert st.tolist() == [3, -1] and h.tolist() == [65, 0] and p.d_count.item() == 8
    assert torch.equal(free, p.d_free)


def test_kv_plan_replayed_in_a_graph_advances_its_own_state(qasr, cuda_device):
    import torch
    n, steps = 7, 150
    p = Pages(torch, 10, 8, 60, seed=5)
    slot, held = [9, 2, 4, 0, 1, 7, 3], [0, 10, 63, 64, 65, 100, 128]
    got = p.plan(qasr, slot, [0] * n, held)
    _check_plan(p, got, slot, [0] * n, held)
    s, h = _ints(slot, torch), _ints(held, torch)
    cu, st = _ints([0] * (n + 1), torch), _ints([0, 0], torch)
    rs, rp = _ints([0] * n, torch), _ints([0] * n, torch)

    def step():
        qasr.kernel_kv_plan(0, _stream(torch), s.data_ptr(), h.data_ptr(), None, n, 10, p.d_table.data_ptr(), 8,
                            p.d_free.data_ptr(), 60, p.d_count.data_ptr(), h.data_ptr(), p.d_count.data_ptr(),
                            cu.data_ptr(), rs.data_ptr(), rp.data_ptr(), n, st.data_ptr())

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for _ in range(steps):
        graph.replay()
    torch.cuda.synchronize()
    for _ in range(steps):
        p.expect(slot, held, [1] * n)
        held = [x + 1 for x in held]
    assert st.tolist() == [0, 0] and h.tolist() == held and p.d_count.item() == len(p.free)
    assert p.d_table.tolist() == p.table and rp.tolist() == [x - 1 for x in held] and rs.tolist() == slot


# ------------------------------------------------------------------------------------ chunk attention
def _swizzle(torch, pool):
    """Logical page rows <-> the kernels' layout (its own inverse)."""
    p, d = torch.arange(PAGE, device=pool.device)[:, None], torch.arange(DIM, device=pool.device)[None, :]
    col = (((d >> 3) ^ (p & 7)) << 3) | (d & 7)
    return torch.gather(pool, pool.dim() - 1, col.expand(pool.shape))


class Chunks:
    """One call's inputs: `lens` is [(positions before, new rows)]."""

    def __init__(self, torch, lens, nq=16, nkv=8, dtype="f16", layers=1, layer=0, seed=1, q_pad=0, out_pad=0, spread=1.5,
                 extra_rows=3, pool_pages=None, fill=0.0):
        self.torch, self.lens, self.nq, self.nkv, self.layers, self.layer = torch, lens, nq, nkv, layers, layer
        self.t = torch.bfloat16 if dtype == "bf16" else torch.float16
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.n, self.slots = len(lens), len(lens) + 2
        total = [a + b for a, b in lens]
        self.max_pages = max(1, max(-(-x // PAGE) for x in total))
        used = sum(-(-x // PAGE) for x in total)
        self.pool_pages = pool_pages or used + 2
        self.rows = sum(b for _, b in lens)
        self.cap = max(1, self.rows + extra_rows)
        order = torch.randperm(self.pool_pages, generator=g, device="cuda")[:used].to(torch.int32)
        self.slot = torch.randperm(self.slots, generator=g, device="cuda")[:self.n].to(torch.int32)
        self.pool = torch.full((self.pool_pages, layers, 2, nkv, PAGE, DIM), fill, dtype=self.t, device="cuda")
        self.table = torch.full((self.slots, self.max_pages), -1, dtype=torch.int32, device="cuda")
        # logical keys and values per request, written through the table
        self.kv = []
        at = 0
        for i, x in enumerate(total):
            np_ = -(-x // PAGE)
            pages = order[at:at + np_]
            at += np_
            self.table[self.slot[i].long(), :np_] = pages
            kv = torch.empty((2, nkv, x, DIM), dtype=self.t, device="cuda").normal_(generator=g)
            self.kv.append(kv)
        self.q = torch.empty((self.cap, nq * DIM + q_pad), dtype=self.t, device="cuda").normal_(0.0, spread, generator=g)
        self.out = torch.full((self.cap, nq * DIM + out_pad), 77.0, dtype=self.t, device="cuda")
        cu = [0]
        for _, b in lens:
            cu.append(cu[-1] + b)
        self.cu, self.kv_len = _ints(cu, torch), _ints(total, torch)
        self.store()

    def store(self):
        """Write self.kv into the pool's pages (what lies behind a request's end stays as it is)."""
        for i, kv in enumerate(self.kv):
            x = kv.shape[2]
            np_ = -(-x // PAGE)
            if not np_:
                continue
            pages = self.table[self.slot[i].long(), :np_].long()
            rows = _swizzle(self.torch, self.pool[pages, self.layer])  # [pages, 2, nkv, 64, 128]
            flat = rows.permute(1, 2, 0, 3, 4).reshape(2, self.nkv, np_ * PAGE, DIM).clone()
            flat[:, :, :x] = kv
            back = flat.view(2, self.nkv, np_, PAGE, DIM).permute(2, 0, 1, 3, 4)
            self.pool[pages, self.layer] = _swizzle(self.torch, back.contiguous())

    def workspace(self, qasr):
        n = qasr.kernel_attention_chunk_workspace(0)
        # any content will do: bytes that read as NaN in every type
        return self.torch.full((n,), 0xff, dtype=self.torch.uint8, device="cuda"), n

    def run(self, qasr, ws=None, out=None, scale=None, stream=None):
        ws, n = ws or self.workspace(qasr)
        out = self.out if out is None else out
        qasr.kernel_attention_chunk(0, _stream(self.torch) if stream is None else stream,
                                    qasr.TYPE_BF16 if self.t == self.torch.bfloat16 else qasr.TYPE_F16, self.q.data_ptr(),
                                    self.q.shape[1], out.data_ptr(), out.shape[1], self.cap, self.pool.data_ptr(),
                                    self.pool_pages, self.table.data_ptr(), self.slots, self.max_pages, self.layers, self.nq,
                                    self.nkv, self.layer, self.slot.data_ptr(), self.cu.data_ptr(), self.kv_len.data_ptr(),
                                    self.n, ws.data_ptr(), n, **({} if scale is None else {"scale": scale}))
        return out

    def check(self, out, scale=DIM ** -0.5, skip=()):
        """Against the formula in 64 bits.  With u half a step of the type, A = sum p|v| / sum p and n keys, an output
        is off by at most
          u|o|            its own rounding
          u A             the probabilities' rounding before the product with V
          4 E A           scores off by E = 128 * 2^-22 * scale * max_t sum_i |q_i k_ti| (f32 products summed in any
                          order, with truncation), which p = e^s and the sum over p each feel at most twice
          n 2^-21 A       the f32 sums over the keys, of p v and of p, and the exponential's last bits
          n 2^-25 max|v|  f16 probabilities below its normal range (the largest probability is at least 1 before
                          the division), and 2^-25 for an output there."""
        torch = self.torch
        u = torch.finfo(self.t).eps / 2
        first, worst = 0, 0.0
        for i, (a, b) in enumerate(self.lens):
            k, v = self.kv[i][0].double(), self.kv[i][1].double()
            G = self.nq // self.nkv
            for r in range(0, b, 1024):
                m = min(1024, b - r)
                q = self.q[first + r:first + r + m, :self.nq * DIM].double().view(m, self.nkv, G, DIM).permute(1, 2, 0, 3)
                s = torch.einsum("gjmd,gtd->gjmt", q, k) * scale
                size = torch.einsum("gjmd,gtd->gjmt", q.abs(), k.abs()) * abs(scale)
                hidden = torch.arange(a + b, device="cuda")[None, :] > (a + r + torch.arange(m, device="cuda"))[:, None]
                s = s.masked_fill(hidden, -torch.inf)
                E = 128 * 2.0 ** -22 * size.masked_fill(hidden, 0.0).amax(-1)
                p = torch.softmax(s, -1)
                o = torch.einsum("gjmt,gtd->gjmd", p, v)
                A = torch.einsum("gjmt,gtd->gjmd", p, v.abs())
                n = a + b
                tol = (u * o.abs() + (u + 4 * E[..., None] + n * 2.0 ** -21) * A) * 1.01
                tol += n * 2.0 ** -25 * v.abs().amax() + 2.0 ** -25
                got = out[first + r:first + r + m, :self.nq * DIM].double().view(m, self.nkv, G, DIM).permute(1, 2, 0, 3)
                bad = ~((got - o).abs() <= tol)
                if skip:
                    keep = torch.tensor([first + r + x not in skip for x in range(m)], device="cuda")
                    bad = bad[:, :, keep]
                assert not bad.any(), (i, r, int(bad.sum()), float((got - o).abs().nan_to_num(9e9).max()), float(tol.max()))
                worst = max(worst, float(((got - o).abs() / tol).nan_to_num(0).max()))
            first += b
        # what no request owns is left alone
        assert (out[self.rows:] == 77).all() and (out[:, self.nq * DIM:] == 77).all()
        return worst


HEADS = [(16, 8), (8, 8), (16, 2), (12, 4), (16, 1), (5, 1)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("nq,nkv", HEADS)
@pytest.mark.parametrize("lens", [
    [(0, 1)], [(63, 1), (64, 1), (0, 2), (65, 3)], [(0, 64)], [(0, 65), (130, 1)], [(100, 13)] * 5,
    [(0, 128), (1, 127), (127, 129)], [(500, 300), (3, 0), (0, 0), (900, 1)],
], ids=["one", "few", "page", "odd", "append", "blocks", "mixed"])
def test_chunk_attention_matches_the_formula(qasr, cuda_device, lens, nq, nkv, dtype):
    import torch
    c = Chunks(torch, lens, nq=nq, nkv=nkv, dtype=dtype, seed=len(lens) + nq)
    ws = c.workspace(qasr)
    out = c.run(qasr, ws=ws)
    qasr.kernel_attention_chunk_check(0, _stream(torch), ws[0].data_ptr())  # waits for the stream
    c.check(out)


@pytest.mark.parametrize("lens", [
    [(4095, 1)], [(0, 2000)], [(3000, 40), (17, 1)], [(i * 7 % 1500, 1) for i in range(200)],
    [(200 * i, 37 * i + 1) for i in range(12)], [(5000, 700)], [(0, 257)] * 9 + [(2222, 1)] * 40,
], ids=["long-token", "prompt", "few-rows-long", "decode-200", "ragged", "chunk-of-long", "prefill-and-decode"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_chunk_attention_long(qasr, cuda_device, lens, dtype):
    import torch
    c = Chunks(torch, lens, dtype=dtype, layers=2, layer=1, q_pad=8, out_pad=24, seed=len(lens))
    out = c.run(qasr)
    torch.cuda.synchronize()
    c.check(out)


@pytest.mark.parametrize("spread,scale", [(30.0, None), (0.0, None), (1.0, 0.5), (1.0, -0.1), (1.0, 0.0)])
def test_chunk_attention_scores(qasr, cuda_device, spread, scale):
    """One-hot softmaxes whose maximum keeps moving, flat ones, and other scales."""
    import torch
    c = Chunks(torch, [(400, 150), (0, 300), (777, 1)], spread=spread, seed=4)
    out = c.run(qasr, scale=scale)
    torch.cuda.synchronize()
    c.check(out, scale=DIM ** -0.5 if scale is None else scale)


def test_chunk_attention_rising_scores(qasr, cuda_device):
    """Every key beats the ones before it by far, so the running maximum is replaced all along."""
    import torch
    c = Chunks(torch, [(700, 200), (1500, 1)], seed=6)
    for kv in c.kv:
        n = kv.shape[2]
        kv[0] = (torch.arange(n, device="cuda") * (8.0 / n))[None, :, None]
    c.store()
    c.q.fill_(1.0)
    out = c.run(qasr)
    torch.cuda.synchronize()
    c.check(out)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("lens", [[(0, 1)], [(70, 1), (0, 3)], [(0, 200)], [(300, 100), (0, 64)], [(1000, 1)]])
def test_chunk_attention_never_uses_what_lies_behind_the_end(qasr, cuda_device, lens, dtype):
    """NaN everywhere in the pool but at the requests' own positions."""
    import torch
    c = Chunks(torch, lens, dtype=dtype, fill=float("nan"), seed=9)
    out = c.run(qasr)
    torch.cuda.synchronize()
    c.check(out)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("which", [0, 1])
def test_chunk_attention_later_positions_do_not_reach_earlier_rows(qasr, cuda_device, which, value):
    """A key or value that is not finite at position p leaves the rows before p as they were."""
    import torch
    c = Chunks(torch, [(90, 200), (0, 40), (300, 1)], seed=10)
    clean = c.run(qasr).clone()
    torch.cuda.synchronize()
    kv = [x.clone() for x in c.kv]
    c.kv[0][which, :, 90 + 150] = value
    c.kv[1][which, :, 39] = value
    c.store()
    out = c.run(qasr)
    torch.cuda.synchronize()
    c.kv = kv
    c.check(out, skip=set(range(150, 200)) | {239})
    assert clean.isfinite().all()
    if which == 1 and value != value:
        assert out[150:200, :c.nq * DIM].isnan().all() and out[239, :c.nq * DIM].isnan().all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("at", [64 + x for x in range(8)] + [127, 130])
def test_chunk_attention_a_key_that_is_not_a_number_shows_in_every_row_that_sees_it(qasr, cuda_device, at, dtype):
    """Whatever column of a tile it stands in: a chunk of two row tiles, a cut decode row and a short chunk."""
    import torch
    c = Chunks(torch, [(0, 150), (1000, 1), (120, 20)], seed=19, dtype=dtype)
    kv = [x.clone() for x in c.kv]
    for x in c.kv:
        x[0, :, at] = float("nan")
    c.store()
    out = c.run(qasr)
    torch.cuda.synchronize()
    seen = set(range(at, 150)) | {150} | {151 + j for j in range(20) if 120 + j >= at}
    for r in seen:
        assert out[r, :2048].isnan().all(), r
    c.kv = kv
    c.check(out, skip=seen)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_chunk_attention_huge_values_at_masked_positions(qasr, cuda_device, dtype):
    """The largest finite values at later positions: a masked probability is exactly 0."""
    import torch
    c = Chunks(torch, [(64, 128), (10, 60)], seed=20, dtype=dtype)
    kv = [x.clone() for x in c.kv]
    for x in c.kv:
        x[1, :, -60:] = torch.finfo(c.t).max
    c.store()
    out = c.run(qasr)
    torch.cuda.synchronize()
    c.kv = kv
    c.check(out, skip=set(range(68, 128)) | set(range(128, 188)))


def test_chunk_attention_rows_that_see_nothing(qasr, cuda_device):
    """More rows than positions: the rows before position 0 are zeros; a request without any position too."""
    import torch
    c = Chunks(torch, [(0, 50), (0, 6), (0, 1)], seed=11)
    c.kv_len = _ints([20, 0, 1], torch)
    out = c.run(qasr)
    torch.cuda.synchronize()
    assert (out[:30, :2048] == 0).all() and (out[50:56, :2048] == 0).all()
    assert torch.equal(out[56, :2048].view(8, 2, 128), c.kv[2][1, :, 0][:, None].expand(8, 2, 128))
    d = Chunks(torch, [(0, 20)], seed=11)
    d.kv, d.q, d.slot, d.table, d.pool = [c.kv[0][:, :, :20].contiguous()], c.q[30:], c.slot[:1], c.table, c.pool
    got = torch.full_like(d.out, 77)
    got[:20] = out[30:50]
    d.check(got)


def test_chunk_attention_device_arrays_out_of_range_stay_inside(qasr, cuda_device):
    """Slots, pages, lengths and row bounds that are wrong are cut back, never followed."""
    import torch
    c = Chunks(torch, [(100, 20), (50, 10), (0, 30)], seed=12, extra_rows=4)
    c.slot[1] = 99
    c.table[c.slot[2].long(), 0] = c.pool_pages + 5
    c.cu = _ints([0, 20, 30, 10**6], torch)
    c.kv_len = _ints([120, 60, 2**31 - 1], torch)
    out = c.run(qasr)
    torch.cuda.synchronize()
    assert (out[20:30, :2048] == 0).all()
    c.lens, c.rows = c.lens[:1], 20
    c.check(torch.cat([out[:20], torch.full_like(out[:3], 77)]))


def test_chunk_attention_offsets_past_32_bits(qasr, cuda_device):
    """A pool of more than 2^32 elements, the requests' pages at its end."""
    import torch
    pages = (1 << 32) // (2 * 8 * PAGE * DIM) + 40
    c = Chunks(torch, [(200, 70), (1000, 1)], seed=13, pool_pages=pages)
    used = int((c.table >= 0).sum())
    old = c.table.clone()
    c.table[old >= 0] = torch.arange(pages - used, pages, device="cuda", dtype=torch.int32)
    c.store()
    out = c.run(qasr)
    torch.cuda.synchronize()
    c.check(out)


def test_chunk_attention_repeats_bit_for_bit_on_other_streams(qasr, cuda_device):
    """The same call twice, and two calls at once on two streams with a workspace each."""
    import torch
    c = Chunks(torch, [(700, 90), (1200, 1), (0, 300)] * 3, seed=14)
    d = Chunks(torch, [(2500, 1)] * 20, seed=15, dtype="bf16")
    a, b = c.run(qasr).clone(), d.run(qasr).clone()
    torch.cuda.synchronize()
    wc, wd = c.workspace(qasr), d.workspace(qasr)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        c.run(qasr, ws=wc, stream=s1.cuda_stream)
        d.run(qasr, ws=wd, stream=s2.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(a, c.out) and torch.equal(b, d.out)


def test_chunk_attention_captured_and_replayed_with_other_lengths(qasr, cuda_device):
    """One graph, the lengths and tables changed between its replays: no length reaches the host."""
    import torch
    c = Chunks(torch, [(40, 60), (300, 1), (0, 200)], seed=16)
    ws = c.workspace(qasr)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        c.run(qasr, ws=ws)
    graph.replay()
    torch.cuda.synchronize()
    c.check(c.out)
    # the second request leaves, the third adds one row only
    c.out.fill_(77)
    c.cu.copy_(_ints([0, 60, 60, 61], torch))
    c.lens, c.rows = [(40, 60), (301, 0), (199, 1)], 61
    graph.replay()
    torch.cuda.synchronize()
    c.check(c.out)


@pytest.mark.parametrize("n", [33, 1000, 1025, 2500])
def test_chunk_attention_many_requests(qasr, cuda_device, n):
    """As many requests as the schedule reads in one, two and several steps, empty ones and chunks among them."""
    import torch
    rng = random.Random(n)
    lens = [(rng.randint(0, 40), rng.choice([0, 1, 1, 1, 2, 5])) for _ in range(n)]
    lens[n // 2] = (300, 200)
    c = Chunks(torch, lens, nq=8, nkv=4, seed=n)
    ws = c.workspace(qasr)
    out = c.run(qasr, ws=ws)
    qasr.kernel_attention_chunk_check(0, _stream(torch), ws[0].data_ptr())
    c.check(out)


def test_chunk_attention_very_many_tiles(qasr, cuda_device):
    """More than 2^22 key tiles in one call (requests that share their pages), where cuts are placed in 64 bits."""
    import torch
    n, ctx = 4200, 8191
    c = Chunks(torch, [(ctx, 1)], seed=18)
    c.n = c.slots = n
    c.table = c.table[c.slot[0].long()].repeat(n, 1)
    c.slot = torch.arange(n, dtype=torch.int32, device="cuda")
    c.cu = torch.arange(n + 1, dtype=torch.int32, device="cuda")
    c.kv_len = torch.full((n,), ctx + 1, dtype=torch.int32, device="cuda")
    c.cap = n
    c.q = c.q[:1].repeat(n, 1)
    out = c.run(qasr, out=torch.full((n, 2048), 77.0, dtype=torch.float16, device="cuda"))
    torch.cuda.synchronize()
    got = torch.full((2, 2048), 77.0, dtype=torch.float16, device="cuda")
    for r in (0, 1, n // 2, n - 1):
        got[0] = out[r]
        c.check(got)
    # every row against the first: two errors of at most u|o| and u A each (with the terms of `check` that are small here),
    # A = sum p|v| / sum p being an average of |v| over 8192 keys, below 1
    first = out[:1].float()
    assert ((out.float() - first).abs() <= 2 * 2.0 ** -11 * 1.1 * (first.abs() + 1)).all()


def test_chunk_attention_small_workspace_is_refused(qasr, cuda_device):
    import torch
    c = Chunks(torch, [(0, 4)])
    ws, n = c.workspace(qasr)
    with pytest.raises(qasr.DecoderError) as e:
        c.run(qasr, ws=(ws, n - 1))
    assert e.value.status == 3


def test_chunk_attention_agrees_with_the_decode_attention(qasr, cuda_device):
    """One row per slot is qasr_kernel_attention's case: both against the same formula, so within two tolerances."""
    import torch
    c = Chunks(torch, [(n - 1, 1) for n in (1, 64, 65, 700, 1500, 4096)], seed=17)
    out = c.run(qasr)
    other = torch.full_like(c.out, 77)
    pos = c.kv_len - 1
    qasr.kernel_attention(0, _stream(torch), c.q.data_ptr(), 2048, other.data_ptr(), c.pool.data_ptr(), c.table.data_ptr(),
                          c.max_pages, 1, 8, 0, c.slot.data_ptr(), pos.data_ptr(), c.n)
    torch.cuda.synchronize()
    c.check(out)
    c.check(other)


# ------------------------------------------------------------------------------------ 4-bit products
class W4:
    def __init__(self, qasr, torch, n_out, k, group, zeros, dtype, rows, seed=1, x_pad=0, o_pad=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.torch, self.n_out, self.k, self.group, self.rows = torch, n_out, k, group, rows
        self.t = torch.bfloat16 if dtype == "bf16" else torch.float16
        self.codes = torch.randint(0, 256, (n_out, k // 2), dtype=torch.uint8, device="cuda", generator=g)
        self.scale = (torch.rand((n_out, k // group), device="cuda", generator=g) * 0.01 + 0.001).to(torch.float16)
        self.zero = torch.randint(0, 16, (n_out, k // group), dtype=torch.uint8, device="cuda", generator=g) if zeros else None
        self.x = torch.empty((rows, k + x_pad), dtype=self.t, device="cuda").normal_(generator=g)
        if x_pad:
            self.x[:, k:] = float("nan")  # behind a row's end
        self.out = torch.full((rows + 1, n_out + o_pad), 77.0, dtype=self.t, device="cuda")
        n = qasr.kernel_w4_packed_bytes(n_out, k, group, zeros)
        self.packed = torch.full((n + 64,), 0xff, dtype=torch.uint8, device="cuda")
        qasr.kernel_pack_w4(0, _stream(torch), self.codes.data_ptr(), self.scale.data_ptr(),
                            self.zero.data_ptr() if zeros else None, n_out, k, group, self.packed.data_ptr())
        assert (self.packed[n:] == 0xff).all()

    def run(self, qasr, accumulate=False):
        qasr.kernel_gemv_w4(0, _stream(self.torch), qasr.TYPE_BF16 if self.t == self.torch.bfloat16 else qasr.TYPE_F16,
                            self.packed.data_ptr(), self.zero is not None, self.n_out, self.k, self.group,
                            self.x.data_ptr(), self.x.shape[1], self.rows, self.out.data_ptr(), self.out.shape[1], accumulate)
        return self.out

    def weight(self):
        torch = self.torch
        u = torch.stack([self.codes & 15, self.codes >> 4], -1).view(self.n_out, self.k).double()
        z = self.zero.double().repeat_interleave(self.group, 1) if self.zero is not None else 8.0
        return (u - z) * self.scale.double().repeat_interleave(self.group, 1)

    def check(self, out, before=None):
        """Exact products, a group's sum in f32 (any order, with truncation), the groups' sums in f32: an output is off by
        its own rounding u|y| and by (group + k / group + 32) steps of 2^-23 of sum |w x|."""
        torch = self.torch
        w, x = self.weight(), self.x[:, :self.k].double()
        y, size = x @ w.t(), x.abs() @ w.abs().t()
        if before is not None:
            y, size = y + before.double(), size + before.double().abs()
        u = torch.finfo(self.t).eps / 2
        tol = u * y.abs() * 1.01 + (self.group + self.k / self.group + 32) * 2.0 ** -23 * size + 2.0 ** -25
        got = out[:self.rows, :self.n_out].double()
        bad = ~((got - y).abs() <= tol)
        assert not bad.any(), (int(bad.sum()), bad.nonzero()[:4].tolist(), float((got - y).abs().max()), float(tol.max()))
        assert (out[self.rows:] == 77).all() and (out[:, self.n_out:] == 77).all()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("n_out,k,group,rows", [
    (1, 32, 32, 1), (16, 64, 64, 1), (17, 96, 32, 2), (15, 160, 32, 9), (128, 128, 128, 8), (1024, 2048, 32, 1),
    (1000, 1984, 64, 3), (2048, 6144, 64, 16), (4096, 2048, 128, 17), (333, 4096, 128, 31), (700, 640, 64, 33),
    (300, 8192, 32, 64), (12288, 2048, 128, 5), (20000, 256, 128, 1), (2500, 1024, 64, 40),
])
def test_w4_matches_the_formula(qasr, cuda_device, n_out, k, group, rows, zeros, dtype):
    import torch
    w = W4(qasr, torch, n_out, k, group, zeros, dtype, rows, seed=n_out + k)
    out = w.run(qasr)
    torch.cuda.synchronize()
    w.check(out)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 12, 50])
def test_w4_strides_and_accumulation(qasr, cuda_device, rows, dtype):
    import torch
    w = W4(qasr, torch, 1111, 1440, 32, True, dtype, rows, x_pad=24, o_pad=3)
    w.check(w.run(qasr))
    before = w.out[:rows, :1111].clone()
    w.run(qasr, accumulate=True)
    torch.cuda.synchronize()
    w.check(w.out, before=before)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 7, 20])
def test_w4_codes_are_exact(qasr, cuda_device, rows, dtype):
    """One-hot rows with scales that are powers of two: every output is one weight, bit for bit."""
    import torch
    w = W4(qasr, torch, 160, 256, 64, True, dtype, rows, seed=5)
    w.scale.copy_(2.0 ** torch.randint(-6, 2, w.scale.shape, device="cuda"))
    qasr.kernel_pack_w4(0, _stream(torch), w.codes.data_ptr(), w.scale.data_ptr(), w.zero.data_ptr(), 160, 256, 64,
                        w.packed.data_ptr())
    for c0 in range(0, 256, rows):
        cols = [(c0 + r) % 256 for r in range(rows)]
        w.x.zero_()
        w.x[torch.arange(rows), cols] = 1.0
        w.run(qasr)
        torch.cuda.synchronize()
        assert torch.equal(w.out[:rows, :160].double(), w.weight()[:, cols].t())


def test_w4_rows_do_not_touch_each_other(qasr, cuda_device):
    """A row of NaN stays its own; rows past the call's last are never read into a result."""
    import torch
    w = W4(qasr, torch, 500, 512, 128, False, "f16", 6, seed=6)
    clean = w.run(qasr).clone()
    w.x[3] = float("nan")
    w.x[5, 7] = float("inf")
    out = w.run(qasr)
    torch.cuda.synchronize()
    assert out[3, :500].isnan().all()
    keep = [0, 1, 2, 4]
    assert torch.equal(out[keep], clean[keep])


def test_w4_captured_and_replayed(qasr, cuda_device):
    import torch
    w = W4(qasr, torch, 2048, 1024, 64, False, "f16", 4, seed=7)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        w.run(qasr)
    for seed in (1, 2):
        w.x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        w.check(w.out)


def test_calls_leave_the_current_device_alone(qasr, cuda_device):
    import torch
    before = torch.cuda.current_device()
    w = W4(qasr, torch, 64, 64, 64, False, "f16", 1)
    w.run(qasr)
    assert torch.cuda.current_device() == before


# ------------------------------------------------------------------------------------ all of them together
@pytest.mark.parametrize("dtype", ["f16"])
def test_a_serving_step_of_all_operators(qasr, cuda_device, dtype):
    """A layer's attention block over several steps as a server runs it: maps and pages, the 4-bit q|k|v product, the
    cache's append, the attention of the chunk, the 4-bit output product added to the residual; first a chunk per
    request, then single tokens, then one request leaves.  Every stage is held to the formula of its own inputs."""
    import torch
    hs, nq, nkv, max_pages, slots, pool_pages = 512, 16, 8, 4, 6, 14
    p = Pages(torch, slots, max_pages, pool_pages, seed=8)
    pool = torch.full((pool_pages, 1, 2, nkv, PAGE, DIM), float("nan"), dtype=torch.float16, device="cuda")
    qkv = W4(qasr, torch, (nq + 2 * nkv) * DIM, hs, 64, True, dtype, 64, seed=1)
    o = W4(qasr, torch, hs, nq * DIM, 128, False, dtype, 64, seed=2)
    qkv.scale.mul_(0.3)
    qasr.kernel_pack_w4(0, _stream(torch), qkv.codes.data_ptr(), qkv.scale.data_ptr(), qkv.zero.data_ptr(), qkv.n_out, hs,
                        64, qkv.packed.data_ptr())
    n_ws = qasr.kernel_attention_chunk_workspace(0)
    ws = torch.empty(n_ws, dtype=torch.uint8, device="cuda")
    cache = {s: torch.empty((2, nkv, 0, DIM), dtype=torch.float16, device="cuda") for s in range(slots)}
    slot, held = [4, 0, 3], [0, 0, 0]
    for new in ([30, 21, 13], [1, 1, 1], [20, 0, 40], [1, 1, 1], [1, 1, 1]):
        d_slot, d_len = _ints(slot, torch), _ints(held, torch)
        rows = sum(new)
        cu, maps, status = _ints([0] * 4, torch), [_ints([0] * rows, torch) for _ in range(2)], _ints([0, 0], torch)
        d_new = _ints(new, torch)
        qasr.kernel_kv_plan(0, _stream(torch), d_slot.data_ptr(), d_len.data_ptr(), d_new.data_ptr(), 3, slots,
                            p.d_table.data_ptr(), max_pages, p.d_free.data_ptr(), pool_pages, p.d_count.data_ptr(),
                            d_len.data_ptr(), p.d_count.data_ptr(), cu.data_ptr(), maps[0].data_ptr(), maps[1].data_ptr(),
                            rows, status.data_ptr())
        p.expect(slot, held, new)
        qkv.rows = rows
        qkv.x = torch.randn((rows, hs), device="cuda").to(torch.float16)
        y = qkv.out = torch.full((rows + 1, qkv.n_out), 77.0, dtype=torch.float16, device="cuda")
        qkv.run(qasr)
        k = y[:rows, nq * DIM:(nq + nkv) * DIM].contiguous()
        v = y[:rows, (nq + nkv) * DIM:].contiguous()
        qasr.kernel_kv_append(0, _stream(torch), k.data_ptr(), v.data_ptr(), pool.data_ptr(), p.d_table.data_ptr(), max_pages,
                              1, nkv, 0, maps[0].data_ptr(), maps[1].data_ptr(), rows)
        att = torch.full((rows + 1, nq * DIM), 77.0, dtype=torch.float16, device="cuda")
        qasr.kernel_attention_chunk(0, _stream(torch), qasr.TYPE_F16, y.data_ptr(), y.shape[1], att.data_ptr(), nq * DIM, rows,
                                    pool.data_ptr(), pool_pages, p.d_table.data_ptr(), slots, max_pages, 1, nq, nkv, 0,
                                    d_slot.data_ptr(), cu.data_ptr(), d_len.data_ptr(), 3, ws.data_ptr(), n_ws)
        o.rows, o.x = rows, att
        o.out = torch.full((rows + 1, hs), 77.0, dtype=torch.float16, device="cuda")
        o.out[:rows] = torch.randn((rows, hs), device="cuda").to(torch.float16)
        resid = o.out[:rows].clone()
        o.run(qasr, accumulate=True)
        torch.cuda.synchronize()
        assert status.tolist() == [0, 0] and p.d_table.tolist() == p.table
        qkv.check(y)
        c = Chunks.__new__(Chunks)
        c.torch, c.t, c.nq, c.nkv, c.rows = torch, torch.float16, nq, nkv, rows
        c.lens = list(zip(held, new))
        c.q, c.kv, first = y[:, :nq * DIM], [], 0
        for i, s in enumerate(slot):
            add = torch.stack([k[first:first + new[i]], v[first:first + new[i]]]).view(2, new[i], nkv, DIM).transpose(1, 2)
            cache[s] = torch.cat([cache[s], add], 2)
            c.kv.append(cache[s])
            first += new[i]
        c.check(att)
        o.x = att[:rows]
        o.check(o.out, before=resid)
        held = d_len.tolist()
        assert held == [a + b for a, b in c.lens]
