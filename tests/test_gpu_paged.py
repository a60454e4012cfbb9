"""The paged-serving operators against plain 64-bit implementations: page planning and
release, cache append, attention of a chunk of new tokens over the paged cache.

Tolerances of the attention, per output element, u = 2^-11 (fp16) or 2^-8 (bf16):
the probabilities are rounded to 16 bits (relative u each) and so is their sum's
counterpart, the output once more (u |o|); fp32 scores of up to 256 products of
magnitude |q||k| scale err below 2^-13 for the inputs used here (|score| < 32), which
moves a probability by as much relatively.  Hence
    |o - ref| <= u |ref| + (2 u + 2^-12) sum_j p_j |v_j| + 2^-24,
times the gate's sigmoid."""
import numpy as np
import pytest
import torch

from thunderllamax_b200 import _lib, ops, paged

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def device():
    ops.require_device()


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------ planning
def plan_model(cached, new, held, table, free, n_free, page, tokens):
    """The planning rule, one request after another, on the host."""
    r, width = table.shape
    table, held = table.copy(), list(held)
    q_start, kv_len, status = [0], [], []
    slots, pos = [-1] * tokens, [-1] * tokens
    top, tok, end = n_free, 0, 0
    for b in range(r):
        c, n, h, st, take = cached[b], new[b], held[b], 0, 0
        if c < 0 or n < 0 or h < 0 or n > tokens:
            st, n, c = 3, (0 if n < 0 or n > tokens else n), 0
        else:
            need = -(-(c + n) // page)
            if need > width or h > width:
                st = 2
            else:
                take = max(0, need - h)
        end += take
        if st == 0 and tok + n > tokens:
            st = 3
        if st == 0 and take > 0 and end > n_free:
            st = 1
        if st == 0:
            for j in range(take):
                top -= 1
                table[b, h + j] = free[n_free - 1 - (end - take + j)]
            held[b] = h + take
        for i in range(n):
            if tok + i < tokens:
                p = c + i
                pos[tok + i] = p
                slots[tok + i] = int(table[b, p // page]) * page + p % page if st == 0 else -1
        tok += n
        q_start.append(min(tok, tokens))
        kv_len.append(c + n if st == 0 else 0)
        status.append(st)
    return dict(table=table, held=held, n_free=top, q_start=q_start, kv_len=kv_len, status=status, slots=slots,
                positions=pos)


def run_plan(cached, new, held, table, free, n_free, page, tokens, in_place=False):
    r, width = table.shape
    pt = paged.PageTable(r, width, len(free), page, table=torch.from_numpy(table.copy()).cuda(), held=i32(held),
                         free=i32(free), n_free=i32([n_free]))
    plan = paged.Plan(r, tokens)
    ho, no = (None, None) if in_place else (torch.empty_like(pt.held), torch.empty_like(pt.n_free))
    for _ in range(1 if in_place else 2):       # a call that updates nothing in place can be made again
        pt.plan(i32(cached), i32(new), plan, held_out=ho, n_free_out=no)
    torch.cuda.synchronize()
    held_t, free_t = (pt.held, pt.n_free) if in_place else (ho, no)
    assert int(pt.ws.buf[:4].view(torch.int32)) == 0
    return dict(table=pt.table.cpu().numpy(), held=held_t.tolist(), n_free=int(free_t), q_start=plan.q_start.tolist(),
                kv_len=plan.kv_len.tolist(), status=plan.status.tolist(), slots=plan.slots.tolist(),
                positions=plan.positions.tolist())


def same_plan(got, want):
    for k in want:
        assert np.array_equal(np.asarray(got[k]), np.asarray(want[k])), k


def plan_inputs(rng, r, page, hi_cached, hi_new, spare, extra_held=0):
    cached = rng.integers(0, hi_cached + 1, r).tolist()
    new = rng.integers(0, hi_new + 1, r).tolist()
    held = [-(-c // page) + int(rng.integers(0, extra_held + 1)) for c in cached]
    width = max(max(held), max(-(-(c + n) // page) for c, n in zip(cached, new))) + 1
    pages = sum(held) + spare
    order = rng.permutation(pages).astype(np.int32)
    table = np.full((r, width), -1, np.int32)
    at = 0
    for b, h in enumerate(held):
        table[b, :h] = order[at:at + h]
        at += h
    free = np.concatenate([order[at:], np.full(at, -7, np.int32)]).tolist()
    return cached, new, held, table, free, pages - at


@pytest.mark.parametrize("r,page,hi_cached,hi_new,spare", [
    (1, 16, 0, 1, 4), (1, 8, 0, 0, 1), (3, 16, 40, 3, 50), (64, 16, 5000, 1, 100), (100, 64, 300, 700, 3000),
    (511, 8, 100, 9, 4000), (512, 16, 100, 9, 4000), (513, 16, 100, 9, 4000), (1500, 256, 3000, 200, 4000),
    (700, 16, 200, 60, 900), (40, 16, 100, 300, 33)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(r, page, hi_cached, hi_new, spare, in_place):
    rng = np.random.default_rng(r * 7 + page)
    cached, new, held, table, free, n_free = plan_inputs(rng, r, page, hi_cached, hi_new, spare, extra_held=2)
    for tokens in (sum(new), sum(new) + 5, max(0, sum(new) - 3)):
        want = plan_model(cached, new, held, table, free, n_free, page, tokens)
        same_plan(run_plan(cached, new, held, table, free, n_free, page, tokens, in_place), want)


def test_plan_refuses_bad_requests_alone():
    cached, new, held = [5, -1, 3, 0, 70, 2], [3, 2, -4, 0, 1, 9], [1, 0, 1, 0, 5, 1]
    table = np.full((6, 4), -1, np.int32)
    table[0, 0], table[2, 0], table[5, 0] = 4, 9, 2
    free = list(range(20, 60))
    want = plan_model(cached, new, held, table, free, 30, 16, 20)
    assert want["status"] == [0, 3, 3, 0, 2, 0]
    same_plan(run_plan(cached, new, held, table, free, 30, 16, 20), want)


def test_plan_release_cycle():
    # requests come and go; every page is always in exactly one place
    rng = np.random.default_rng(3)
    r, width, pages, page = 37, 12, 200, 16
    pt = paged.PageTable(r, width, pages, page)
    lens = np.zeros(r, np.int64)
    for step in range(12):
        new = rng.integers(0, 40, r)
        plan = pt.plan(i32(lens.tolist()), i32(new.tolist()), paged.Plan(r, int(new.sum())))
        ok = plan.status.cpu().numpy() == 0
        lens = np.where(ok, lens + new, lens)
        back = rng.random(r) < 0.3              # rejected drafts: shorter, the pages stay held
        lens = np.where(back, np.maximum(lens - 5, 0), lens)
        done = (rng.random(r) < 0.25) | (lens > (width - 3) * page)
        pt.release(i32(done.astype(int).tolist()))
        lens = np.where(done, 0, lens)
        table, held, n_free = pt.table.cpu().numpy(), pt.held.cpu().numpy(), int(pt.n_free)
        used = [table[b, j] for b in range(r) for j in range(held[b])]
        assert sorted(used + pt.free[:n_free].tolist()) == list(range(pages))
        assert all((table[b, held[b]:] == -1).all() for b in range(r))


# -------------------------------------------------------------------- append
def quantise(x):
    """The int8 rule in 64 bits around its fp32 / fp16 roundings: x [..., d] float32."""
    g = x.reshape(*x.shape[:-1], -1, 32).astype(np.float32)
    m = np.abs(g).max(-1)
    s = np.where(m > 0, m * np.float32(1 / 127), np.float32(1e-8)).astype(np.float16)
    with np.errstate(divide="ignore", invalid="ignore"):
        d = g / s.astype(np.float32)[..., None]
    q = np.rint(np.fmin(np.fmax(d, np.float32(-127)), np.float32(127))) + 128
    return q.reshape(x.shape).astype(np.uint8), s


@pytest.mark.parametrize("hd,heads,page", [(256, 4, 64), (128, 8, 16), (64, 3, 8)])
@pytest.mark.parametrize("x_dtype,cache", [(F16, F16), (BF16, BF16), (torch.float32, F16), (torch.float32, BF16),
                                           (F16, "int8"), (BF16, "int8"), (torch.float32, "int8")])
@pytest.mark.parametrize("tokens", [1, 5, 333])
def test_append(hd, heads, page, x_dtype, cache, tokens):
    g = torch.Generator(device="cuda").manual_seed(tokens + hd)
    pages = tokens // page + 3
    store = paged.PagedCache.empty(pages, page, heads, hd, cache)
    for t in (store.k, store.v):
        t.fill_(7)
    rows = torch.randn((tokens, 2, heads + 1, hd), generator=g, device="cuda").to(x_dtype)   # strided rows
    rows[0, 0, 0, :32] = 0                        # an all-zero int8 group
    rows[tokens // 2, 1, heads - 1] *= 1e-9
    k, v = rows[:, 0, :heads], rows[:, 1, 1:]
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens].to(torch.int32)
    if tokens > 4:
        slots[1], slots[3] = -1, pages * page      # outside the pool: skipped
    store.append(k, v, slots)
    torch.cuda.synchronize()
    want_k, want_v = store.k.clone().fill_(7), store.v.clone().fill_(7)
    if cache == "int8":
        want_ks, want_vs = torch.zeros_like(store.k_scale), torch.zeros_like(store.v_scale)
    for t, s in enumerate(slots.tolist()):
        if not 0 <= s < pages * page:
            continue
        at = (s // page, slice(None), s % page)
        if cache == "int8":
            for x, c, sc in ((k, want_k, want_ks), (v, want_v, want_vs)):
                q, scale = quantise(x[t].float().cpu().numpy())
                c[at], sc[at] = torch.from_numpy(q).cuda(), torch.from_numpy(scale).cuda()
        else:
            want_k[at], want_v[at] = k[t].to(cache), v[t].to(cache)
    assert torch.equal(store.k, want_k) and torch.equal(store.v, want_v)
    if cache == "int8":
        assert torch.equal(store.k_scale, want_ks) and torch.equal(store.v_scale, want_vs)


# ----------------------------------------------------------------- attention
class Batch:
    """Requests with random pages; what no token wrote is NaN (16-bit caches) or has NaN
    scales (int8), and the pages of no request are NaN throughout."""

    def __init__(self, new, kv, heads, kv_heads, hd, cache, page, seed=0, gate=False, nhd=False, amp=1.0, stale=True,
                 pages_apart=None):
        g = torch.Generator(device="cuda").manual_seed(seed + 11)
        self.new, self.kv, self.heads, self.kv_heads, self.hd, self.page = new, kv, heads, kv_heads, hd, page
        need = [-(-t // page) for t in kv]
        pages, width = sum(need) + 2, max(max(need), 1)
        self.dtype = F16 if cache == "int8" else cache
        self.order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
        self.table = torch.full((len(kv), width + 1), -1, dtype=torch.int32, device="cuda")[:, :width]
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = self.order[at:at + n]
            at += n
        shape = (pages, kv_heads, page, hd)
        if pages_apart:
            flat = torch.empty(pages_apart * pages, dtype=self.dtype, device="cuda")
            k, v = (flat[o:].as_strided(shape, (pages_apart, page * hd, hd, 1)) for o in (0, kv_heads * page * hd))
            self.store = paged.PagedCache(k, v)
        elif nhd:
            made = [t.transpose(1, 2).contiguous().transpose(1, 2) if t is not None else None for t in
                    vars(paged.PagedCache.empty(pages, page, kv_heads, hd, cache)).values()
                    if torch.is_tensor(t)]
            self.store = paged.PagedCache(*made)
        else:
            self.store = paged.PagedCache.empty(pages, page, kv_heads, hd, cache)
        s = self.store
        nan = float("nan")
        if cache == "int8":
            for c, sc in ((s.k, s.k_scale), (s.v, s.v_scale)):
                c.copy_(torch.randint(1, 256, shape, dtype=torch.uint8, generator=g, device="cuda"))
                sc.fill_(nan if stale else 1.0)
        else:
            s.k.fill_(nan if stale else 1.0)
            s.v.fill_(nan if stale else 1.0)
        for b, t in enumerate(kv):
            for i in range(need[b]):
                p, n = int(self.table[b, i]), min(page, t - i * page)
                if cache == "int8":
                    for sc in (s.k_scale, s.v_scale):
                        sc[p, :, :n] = (torch.rand((kv_heads, n, hd // 32), generator=g, device="cuda") * 0.02 + 0.01) * amp
                else:
                    for c in (s.k, s.v):
                        c[p, :, :n] = torch.randn((kv_heads, n, hd), generator=g, device="cuda").to(cache) * amp
        tokens = sum(new)
        wide = torch.randn((tokens, heads + 2, hd), generator=g, device="cuda").to(self.dtype)
        self.q = wide[:, 1:1 + heads]            # strided rows
        self.gate = torch.randn((tokens, heads, 2 * hd), generator=g, device="cuda").to(self.dtype)[..., hd:] if gate else None
        self.q_start = i32([0] + np.cumsum(new).tolist())
        self.kv_len = i32(kv)
        self.scale = hd ** -0.5

    def rows(self, b, h):
        """K and V of request b, head h, in 64 bits."""
        t = self.kv[b]
        ids = self.table[b, :-(-t // self.page)].long()
        out = []
        for c, sc in ((self.store.k, self.store.k_scale), (self.store.v, self.store.v_scale)):
            x = c[ids, h].double()
            if sc is not None:
                x = ((x - 128) * sc[ids, h].double().repeat_interleave(32, -1)).half().double()
            out.append(x.reshape(-1, self.hd)[:t])
        return out

    def reference(self):
        """(values, bound without the gate's factor) of every row, in 64 bits."""
        u = 2.0 ** -11 if self.dtype == F16 else 2.0 ** -8
        out = torch.zeros((sum(self.new), self.heads, self.hd), dtype=torch.float64, device="cuda")
        tol = torch.full_like(out, 2.0 ** -24)
        g, at = self.heads // self.kv_heads, 0
        for b, n in enumerate(self.new):
            t = self.kv[b]
            if n and t:
                key = torch.arange(t, device="cuda")
                seen = key[None, :] <= (t - n + torch.arange(n, device="cuda"))[:, None]
                some = seen.any(1)
                for h in range(self.heads):
                    k, v = self.rows(b, h // g)
                    s = (self.q[at:at + n, h].double() @ k.T) * self.scale
                    s = s.masked_fill(~seen, float("-inf"))
                    p = torch.softmax(torch.where(some[:, None], s, torch.zeros_like(s)), -1) * seen
                    # a key that a row does not see has no part in it, whatever its values
                    clean = torch.where(seen.all(0)[:, None] | v.isfinite(), v, torch.zeros_like(v))
                    o = p @ clean
                    out[at:at + n, h] = o
                    tol[at:at + n, h] += u * o.abs() + (2 * u + 2.0 ** -12) * (p @ clean.abs())
            at += n
        if self.gate is not None:
            sg = torch.sigmoid(self.gate.double())
            out, tol = out * sg, tol * sg + 2.0 ** -24 + 2.0 ** -18 * out.abs()
        return out, tol

    def attend(self, **kw):
        attn = paged.PagedAttention(self.heads, self.kv_heads, self.hd)
        args = dict(gate=self.gate, scale=self.scale, max_new=max(self.new + [1]))
        args.update(kw)
        a, b = (attn(self.store, self.table, self.q_start, self.kv_len, self.q, **args) for _ in range(2))
        torch.cuda.synchronize()
        assert attn.error() == 0
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))        # the same bits every time
        return a

    def check(self, **kw):
        got = self.attend(**kw)
        ref, tol = self.reference()
        bad = ((got.double() - ref).abs() <= tol).logical_not()
        assert not bad.any(), (int(bad.sum()), float(((got.double() - ref).abs() / tol).nan_to_num(1e9).max()),
                               bad.nonzero()[:4].tolist())
        return got


HEADS = [(24, 4, 256), (32, 8, 128), (8, 8, 64), (16, 1, 128), (12, 2, 64), (2, 2, 256)]
CACHES = [F16, BF16, "int8"]


@pytest.mark.parametrize("heads,kv_heads,hd", HEADS)
@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("page", [8, 64, 256])
def test_attention_decode(heads, kv_heads, hd, cache, page):
    kv = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 200, 511, 700, 1025]
    Batch([1] * len(kv), kv, heads, kv_heads, hd, cache, page, gate=page == 64).check()


@pytest.mark.parametrize("heads,kv_heads,hd", HEADS + [(128, 1, 64), (96, 4, 128)])
@pytest.mark.parametrize("cache", CACHES)
def test_attention_ragged(heads, kv_heads, hd, cache):
    # nothing new, single tokens, verify rows, chunks, cached and not, and a refused request
    new = [0, 1, 11, 3, 64, 200, 1, 21, 22, 129, 0, 5, 2]
    kv = [40, 1, 150, 3, 64, 333, 0, 300, 22, 700, 0, 70, 0]
    Batch(new, kv, heads, kv_heads, hd, cache, 16, seed=5, gate=hd == 256).check()


@pytest.mark.parametrize("cache", CACHES)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("n,kv", [(1, 1), (2, 2), (16, 16), (17, 80), (100, 100), (257, 1000), (500, 501)])
def test_attention_one_request(cache, hd, n, kv):
    Batch([n], [kv], 8, 2, hd, cache, 32, seed=n, gate=True).check()


def test_attention_rows_without_keys():
    # more new rows than keys: the first rows see nothing and are 0, the later ones the keys there are
    for new, kv in (([5], [3]), ([40, 3], [2, 0]), ([130], [64])):
        b = Batch(new, kv, 6, 1, 128, BF16, 16)
        got = b.check()
        assert (got[: new[0] - kv[0]] == 0).all()


@pytest.mark.parametrize("cache", [F16, "int8"])
def test_attention_long(cache):
    for n in (1, 11):
        Batch([n], [20011], 24, 4, 256, cache, 64, seed=n, gate=True).check()


@pytest.mark.parametrize("hd,cache", [(256, "int8"), (128, BF16), (64, F16)])
def test_attention_many_requests(hd, cache):
    rng = np.random.default_rng(hd)
    kv = rng.integers(1, 400, 300).tolist()
    new = [min(t, int(x)) for t, x in zip(kv, rng.integers(0, 3, 300))]
    Batch(new, kv, 8, 2, hd, cache, 16, seed=1).check()


def test_attention_reused_workspace():
    # one workspace, changing lengths: nothing of an earlier call is left in a later one
    attn = paged.PagedAttention(8, 2, 128)
    attn.ws.buf[256:].fill_(0xFF)
    for i, (new, kv) in enumerate([([1, 1], [900, 64]), ([1, 1], [70, 65]), ([40, 2], [900, 300]), ([1, 1], [129, 1]),
                                   ([3, 33], [66, 500]), ([1, 1], [65, 2000])]):
        b = Batch(new, kv, 8, 2, 128, F16, 16, seed=i)
        got = attn(b.store, b.table, b.q_start, b.kv_len, b.q)
        ref, tol = b.reference()
        assert ((got.double() - ref).abs() <= tol).all(), i


def test_attention_peaked_scores():
    # one key dominates each row, and the running maximum keeps growing along the keys
    for hd, cache, n in ((256, F16, 1), (128, BF16, 70), (64, F16, 300)):
        b = Batch([n], [900], 4, 2, hd, cache, 16, seed=2)
        ramp = torch.linspace(0.1, 1.5, 900, device="cuda")
        for i in range(900):
            p = int(b.table[0, i // 16])
            b.store.k[p, :, i % 16] *= ramp[i]
        b.q *= 3
        b.check()


@pytest.mark.parametrize("n", [1, 4, 90])
def test_attention_future_rows_do_not_leak(n):
    # a later token of the chunk with NaN or infinite K / V changes no earlier row, and makes its own rows NaN
    for hd, cache in ((256, F16), (128, BF16), (64, "int8")):
        b = Batch([n], [n + 70], 4, 2, hd, cache, 16, seed=4, stale=False)
        clean = b.attend()
        last = n + 69
        page, off = int(b.table[0, last // 16]), last % 16
        if cache == "int8":
            b.store.k_scale[page, :, off] = float("nan")
            b.store.v_scale[page, 0, off] = float("inf")
        else:
            b.store.k[page, :, off] = float("nan")
            b.store.v[page, 0, off, 3] = float("inf")
            b.store.v[page, 1, off] = float("nan")
        got = b.attend()
        assert torch.equal(got[: n - 1], clean[: n - 1])
        assert got[n - 1].isnan().all()


def test_attention_infinite_value_reaches_its_rows():
    # an infinite V element that a row sees shows in that row and dim only
    b = Batch([40], [130], 4, 1, 128, F16, 16, seed=6, stale=False)
    clean = b.attend()
    i = 110                                        # seen by rows 20 ..
    b.store.v[int(b.table[0, i // 16]), 0, i % 16, 5] = float("inf")
    got = b.attend()
    assert torch.equal(got[:20], clean[:20])
    assert (got[20:, :, 5] == float("inf")).all()
    rest = [d for d in range(128) if d != 5]
    assert torch.equal(got[20:][..., rest], clean[20:][..., rest])


def test_attention_layouts():
    for cache in CACHES:
        Batch([1, 30], [77, 200], 8, 2, 128, cache, 16, nhd=True).check()


def test_attention_offsets_past_32_bits():
    Batch([1, 40], [33, 70], 4, 2, 64, F16, 16, pages_apart=1 << 29).check()


def test_attention_bad_pages_are_empty():
    # a page id outside the pool reads as zero rows, not as memory
    b = Batch([1], [64], 2, 1, 64, F16, 16, stale=False)
    b.table[0, 1], b.table[0, 2] = -5, 1 << 30
    got = b.attend()
    assert got.isfinite().all()


def test_attention_max_new_and_padding_rows():
    # rows past q_start[-1] and rows past max_new are not written
    b = Batch([3, 1], [50, 20], 4, 2, 128, F16, 16)
    q = torch.cat([b.q, b.q[:2]])
    out = torch.full_like(q, 7.0)
    attn = paged.PagedAttention(4, 2, 128)
    attn(b.store, b.table, b.q_start, b.kv_len, q, out=out, max_new=3)
    ref, tol = b.reference()
    assert ((out[:4].double() - ref).abs() <= tol).all() and (out[4:] == 7).all()


def test_attention_other_stream_and_graph():
    b = Batch([1, 17, 2], [300, 500, 40], 24, 4, 256, "int8", 64)
    want = b.attend()
    attn = paged.PagedAttention(24, 4, 256)
    side = torch.cuda.Stream()
    out = torch.zeros_like(want)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        attn(b.store, b.table, b.q_start, b.kv_len, b.q, out=out)
    side.synchronize()
    assert torch.equal(out, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attn(b.store, b.table, b.q_start, b.kv_len, b.q, out=out)
    b.kv_len[0] = 123
    b.kv[0] = 123
    graph.replay()
    torch.cuda.synchronize()
    ref, tol = b.reference()
    assert ((out.double() - ref).abs() <= tol).all()


def test_step_of_plan_append_attention():
    # prompts in chunks, then single tokens, through planned pages: the same as one dense pass
    hd, heads, kv_heads, page = 128, 8, 2, 16
    g = torch.Generator(device="cuda").manual_seed(0)
    lens = [90, 37, 1]
    k, v, q = ([torch.randn((t, h, hd), generator=g, device="cuda").to(F16) for t in lens]
               for h in (kv_heads, kv_heads, heads))
    pt = paged.PageTable(3, 8, 20, page)
    store = paged.PagedCache.empty(20, page, kv_heads, hd, F16)
    attn = paged.PagedAttention(heads, kv_heads, hd)
    done, outs = [0, 0, 0], [[], [], []]
    for step in ([50, 20, 1], [38, 16, 0], [1, 1, 0], [1, 0, 0]):
        plan = pt.plan(i32(done), i32(step), paged.Plan(3, sum(step)))
        take = lambda x: torch.cat([x[b][done[b]:done[b] + n] for b, n in enumerate(step)])
        store.append(take(k), take(v), plan.slots)
        o = attn(store, pt.table, plan.q_start, plan.kv_len, take(q), max_new=max(step))
        assert plan.status.tolist() == [0, 0, 0]
        at = 0
        for b, n in enumerate(step):
            outs[b].append(o[at:at + n])
            at += n
            done[b] += n
    assert done == lens
    for b, t in enumerate(lens):
        for h in range(heads):
            kk, vv = k[b][:, h // 4].double(), v[b][:, h // 4].double()
            s = (q[b][:, h].double() @ kk.T) * hd ** -0.5
            s = s.masked_fill(torch.ones(t, t, device="cuda").triu(1).bool(), float("-inf"))
            p = torch.softmax(s, -1)
            ref, u = p @ vv, 2.0 ** -11
            tol = u * ref.abs() + (2 * u + 2.0 ** -12) * (p @ vv.abs()) + 2.0 ** -24
            assert ((torch.cat(outs[b])[:, h].double() - ref).abs() <= tol).all()


# ------------------------------------------------------------------ refusals
def test_front_end_refusals():
    b = Batch([1], [20], 4, 2, 128, F16, 16)
    attn = paged.PagedAttention(4, 2, 128)
    with pytest.raises(_lib.TLXError):
        attn(b.store, b.table, b.q_start, b.kv_len, b.q.to(BF16))
    with pytest.raises(_lib.TLXError):
        attn(b.store, b.table.long(), b.q_start, b.kv_len, b.q)
    with pytest.raises(_lib.TLXError):
        attn(b.store, b.table, b.q_start[:1], b.kv_len, b.q)
    with pytest.raises(_lib.TLXError):
        attn(b.store, b.table, b.q_start, b.kv_len, b.q[..., :64])
    with pytest.raises(_lib.TLXError):
        paged.PagedAttention(8, 2, 128)(b.store, b.table, b.q_start, b.kv_len, b.q)
    with pytest.raises(_lib.TLXError):
        paged.PagedAttention(5, 2, 128)
    with pytest.raises(_lib.TLXError):
        paged.PagedCache(b.store.k, b.store.v.to(BF16))
    with pytest.raises(_lib.TLXError):
        paged.PagedCache(b.store.k.to(torch.uint8), b.store.v.to(torch.uint8))
    with pytest.raises(_lib.TLXError):
        b.store.append(b.q, b.q, b.kv_len)
    with pytest.raises(_lib.TLXError):
        b.store.append(b.store.k[0], b.store.v[0], b.kv_len[:0])
    odd = torch.zeros((2, 2, 16, 132), dtype=F16, device="cuda")[..., 1:129]     # rows off 16 bytes
    with pytest.raises(_lib.TLXError):
        paged.PagedCache(odd, odd).append(b.store.k[0, :, :2].transpose(0, 1), b.store.v[0, :, :2].transpose(0, 1),
                                          i32([0, 1]))
    with pytest.raises(_lib.TLXError):
        paged.PageTable(2, 4, 8, 16).plan(i32([0, 0, 0]), i32([1, 1, 1]), paged.Plan(3, 3))
    with pytest.raises(_lib.TLXError):
        paged.PageTable(2, 4, 8, 12).plan(i32([0, 0]), i32([1, 1]), paged.Plan(2, 2))
