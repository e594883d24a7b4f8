"""The paged cache's operators in turn, as a serving loop calls them: prompts with rotary
positions written to their pages, read back for a second turn's attention, decode steps
that append and attend, a page given back and taken by another sequence; the same as one
captured graph, on streams and threads, and on pools whose rows lie far apart."""

import math

import numpy as np
import pytest

from oracle import paged as ref
from tests._helpers import to_np
from tests.test_gpu_paged_cache import host_rows, raw, types
from tests.test_gpu_paged_decode import check, gathered

pytestmark = pytest.mark.gpu


class _Loop:
    def __init__(self, device, name, held, B, Hq, Hkv, D, page, N, seed=0):
        import torch
        from probjax_amd.attention import PagedCache

        self.device, self.name, self.dtype = device, name, types()[name]
        self.B, self.Hq, self.Hkv, self.D, self.page, self.N = B, Hq, Hkv, D, page, N
        self.gen = torch.Generator(device=device).manual_seed(seed)
        self.table = torch.full((B, N), -1, dtype=torch.int32, device=device)
        self.free = list(np.random.default_rng(seed).permutation(B * N))
        self.cache = PagedCache.allocate(B * N, page, Hkv, D, page_table=self.table, dtype=types()[held])
        self.lengths = torch.zeros(B, dtype=torch.int32, device=device)

    def qkv(self, T):
        import torch

        return [torch.randn((self.B, T, h, self.D), generator=self.gen, device=self.device).to(self.dtype)
                for h in (self.Hq, self.Hkv, self.Hkv)]

    def reserve(self, more):
        """Pages for ``more[b]`` further keys of every sequence."""
        for b, n in enumerate((self.lengths.cpu() + more).tolist()):
            for i in range(-(-n // self.page)):
                if self.table[b, i] < 0 and i * self.page >= self.lengths[b] // self.page * self.page:
                    self.table[b, i] = int(self.free.pop())

    def turned(self, q, k):
        import torch
        from probjax_amd.attention import rotary

        T = q.shape[1]
        return rotary(q, k, (self.lengths[:, None] + torch.arange(T, device=self.device))[..., None])

    def append(self, k, v, count=None):
        from probjax_amd.attention import write_pages

        self.lengths = write_pages(self.cache, k, v, kv_lengths=self.lengths, new_lengths=count)

    def attend(self, q):
        from probjax_amd.attention import paged_decode

        import torch

        got, lse = paged_decode(q, self.cache, kv_lengths=self.lengths, return_lse=True)
        torch.cuda.synchronize()
        k, v, there = gathered(self.cache, self.table.cpu().numpy(), None)
        want = ref.paged_decode(to_np(q), np.nan_to_num(k), np.nan_to_num(v), there, self.lengths.cpu().numpy(),
                                1.0 / math.sqrt(self.D))
        check(got, lse, want, self.dtype, self.D, k.shape[1])
        return got


@pytest.mark.parametrize("name,held,B,Hq,Hkv,D,page,prompt", [
    ("bf16", "bf16", 3, 8, 2, 64, 16, 150), ("bf16", "e4m3", 3, 8, 2, 128, 16, 700), ("f16", "e4m3", 2, 6, 3, 80, 20, 90),
    ("f32", "f32", 2, 4, 4, 64, 7, 60), ("f32", "e4m3", 2, 4, 1, 64, 32, 1500),
])
def test_a_serving_loop(device, name, held, B, Hq, Hkv, D, page, prompt):
    import torch
    from probjax_amd import masks
    from probjax_amd.attention import flex_attention, read_pages

    loop = _Loop(device, name, held, B, Hq, Hkv, D, page, -(-(prompt + 60) // page))
    count = torch.tensor([prompt - 17 * b for b in range(B)], dtype=torch.int32, device=device)
    q, k, v = loop.qkv(prompt)
    q, k = loop.turned(q, k)
    loop.reserve(count.cpu())
    loop.append(k, v, count)
    print("prompts", flush=True)
    assert loop.lengths.tolist() == count.tolist()
    back = read_pages(loop.cache, kv_lengths=loop.lengths, length=prompt, dtype=loop.dtype)
    for x, y in zip((k, v), back):
        want = to_np(x).astype(np.float64)
        if held == "e4m3":
            want = ref.decode(*ref.encode(want, name))
        for b in range(B):
            n = int(count[b])
            assert torch.equal(y[b, :n].cpu(), torch.from_numpy(want[b, :n]).to(loop.dtype)) and not y[b, n:].any()
    print("a second turn, of one sequence's new tokens over what it has", flush=True)
    q, k, v = loop.qkv(9)
    q, k = loop.turned(q, k)
    loop.reserve(torch.full((B,), 9))
    loop.append(k, v)
    got = loop.attend(q)
    for b in range(B):
        n = int(loop.lengths[b])
        keys, values = read_pages(loop.cache, kv_lengths=loop.lengths, length=n, dtype=loop.dtype)
        other = flex_attention(q[b:b + 1], keys[b:b + 1], values[b:b + 1], mask=masks.CausalFromBottomRightMask(9, n),
                               enable_gqa=True)
        torch.cuda.synchronize()
        # (each off by a half step of sum p|v| <= max|v| < 8 and of itself, or by float32 sums)
        off = 4 * 8 * max(torch.finfo(loop.dtype).eps / 2, 2.0 ** -13)
        assert (other[0].float() - got[b].float()).abs().max() <= off
    print("steps", flush=True)
    for step in range(4):
        q, k, v = loop.qkv(1)
        q, k = loop.turned(q, k)
        loop.reserve(torch.ones(B, dtype=torch.int32))
        loop.append(k, v)
        loop.attend(q)
        if step == 1:  # the first page of one sequence is the next page of another
            loop.free.append(int(loop.table[0, 0]))
            loop.table[0, 0] = -1
        if step == 2:
            loop.lengths[1] = loop.lengths[1] // page * page  # the last keys dropped, their page too
            i = int(loop.lengths[1]) // page
            if loop.table[1, i] >= 0:
                loop.free.append(int(loop.table[1, i]))
                loop.table[1, i] = -1


@pytest.mark.parametrize("name,held,B,room", [("bf16", "e4m3", 3, 2000), ("f16", "f16", 2, 200), ("f32", "e4m3", 70, 1200)])
def test_a_captured_step(device, name, held, B, room):
    """Append, attend and read back as one graph; the lengths grow in it.  Every replay
    against the eager step on a copy of the cache."""
    import torch
    from probjax_amd.attention import PagedCache, paged_decode, read_pages, write_pages

    dtype, Hq, Hkv, D, page = types()[name], 8, 2, 64, 16
    N = room // page
    gen = torch.Generator(device=device).manual_seed(3)

    def make():
        table = torch.arange(B * N, dtype=torch.int32, device=device).view(B, N).flip(1).contiguous()
        cache = PagedCache.allocate(B * N, page, Hkv, D, page_table=table, dtype=types()[held])
        for t in (cache.k, cache.v):
            t.view(torch.uint8).zero_()
        if held == "e4m3":
            cache.k_exponents.fill_(120), cache.v_exponents.fill_(120)
        return cache

    caches, lengths = [make(), make()], [torch.zeros(B, dtype=torch.int32, device=device) for _ in range(2)]
    q, k, v = (torch.zeros((B, 2, h, D), dtype=dtype, device=device) for h in (Hq, Hkv, Hkv))

    def step(i):
        lengths[i].copy_(write_pages(caches[i], k, v, kv_lengths=lengths[i]))
        o, lse = paged_decode(q, caches[i], kv_lengths=lengths[i], return_lse=True)
        return [o, lse, *read_pages(caches[i], kv_lengths=lengths[i], length=40, dtype=dtype)]

    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        step(0)
    torch.cuda.current_stream(device).wait_stream(side)
    torch.cuda.synchronize()
    lengths[0].zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(0)
    lengths[0].copy_(torch.arange(B) % 5 * (room // 6))
    lengths[1].copy_(lengths[0])
    for rep in range(5):
        print("replay", rep, flush=True)
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=gen, device=device).to(dtype))
        x = torch.randn((300, 300), generator=gen, device=device)
        (x @ x).sum().item()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        want = step(1)
        torch.cuda.synchronize()
        for i, (a, b) in enumerate(zip(got, want)):
            assert torch.equal(a, b), (rep, i)
        assert torch.equal(lengths[0], lengths[1])
        assert np.array_equal(raw(caches[0].k), raw(caches[1].k)) and np.array_equal(raw(caches[0].v), raw(caches[1].v))


def test_two_graphs_with_one_workspace(device):
    """Two captured steps of different sequences whose calls were given the same
    workspace, replayed in turn."""
    import torch
    from probjax_amd.attention import PagedCache
    from probjax_amd.hip_attention import paged_decode

    B, S, Hq, Hkv, D = 2, 3000, 8, 2, 128
    gen = torch.Generator(device=device).manual_seed(4)
    ws = torch.empty(32 << 20, dtype=torch.uint8, device=device)
    sets, graphs = [], []
    for i in range(2):
        q, k, v = (torch.randn(s, generator=gen, device=device).to(torch.bfloat16)
                   for s in ((B, 1, Hq, D), (B, S, Hkv, D), (B, S, Hkv, D)))
        L = torch.tensor([S - 100 * i, 77 + i], dtype=torch.int32, device=device)
        sets.append((q, PagedCache(k, v), L))
    want = [paged_decode(q, c, sm_scale=0.1, kv_lengths=L, return_lse=True) for q, c, L in sets]
    torch.cuda.synchronize()
    for q, c, L in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = paged_decode(q, c, sm_scale=0.1, kv_lengths=L, return_lse=True, workspace=ws)
        graphs.append((g, out))
    for rep in range(4):
        ws.fill_(0xff)
        for g, out in graphs[::1 - 2 * (rep % 2)]:
            g.replay()
        torch.cuda.synchronize()
        for (_, got), w in zip(graphs, want):
            assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])


def test_streams_and_threads_at_once(device):
    """Calls on the same cache from four host threads, each on a stream of its own."""
    import threading

    import torch
    from probjax_amd.attention import paged_decode, read_pages, write_pages

    loops = [_Loop(device, "bf16", "e4m3", 3, 8, 2, 64, 16, 80, seed=i) for i in range(4)]
    for loop in loops:
        loop.reserve(torch.tensor([1200, 40, 333]))
        _, k, v = loop.qkv(1200)
        loop.append(k, v, torch.tensor([1200, 40, 333], device=device))
    new = [loop.qkv(3) for loop in loops]
    shared = loops[0].cache
    shared_q, shared_lengths = new[0][0], loops[0].lengths.clone()

    def work(loop, x):
        k, v = read_pages(loop.cache, kv_lengths=loop.lengths, length=50)
        lengths = write_pages(loop.cache, x[1], x[2], kv_lengths=loop.lengths - 3)  # the same slots every time
        return [paged_decode(x[0], loop.cache, kv_lengths=lengths), paged_decode(x[0], shared, kv_lengths=shared_lengths // 2),
                paged_decode(shared_q, shared, kv_lengths=shared_lengths // 3), k, v]

    for _ in range(2):  # (so that the read sees what was written)
        want = [work(loop, x) for loop, x in zip(loops, new)]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def run(i):
        try:
            s = torch.cuda.Stream(device)
            with torch.cuda.stream(s):
                for _ in range(3):
                    res = work(loops[i], new[i])
                s.synchronize()
            got[i] = res
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for i in range(4):
        for j, (a, b) in enumerate(zip(got[i], want[i])):
            assert torch.equal(a, b), (i, j)


@pytest.mark.parametrize("held", ["bf16", "e4m3"])
@pytest.mark.parametrize("axis", ["page", "token", "head"])
def test_rows_far_apart(device, held, axis):
    """Pools whose pages, tokens or heads lie so far apart that offsets pass 32 bits, and
    new rows as far apart: as on pools that lie close together, bit for bit."""
    import torch
    from probjax_amd.attention import PagedCache, paged_decode, read_pages, write_pages

    B, Hq, H, D, page = 2, 6, 3, 64, 8
    N = 200  # more than a workgroup takes whole
    pages, dtype = 2 * N, types()[held]
    gen = torch.Generator(device=device).manual_seed(5)
    rng = np.random.default_rng(5)
    table = torch.from_numpy(rng.permutation(pages)[:B * N].reshape(B, N).astype(np.int32)).to(device)
    step = {"page": 2 ** 32 // (pages - 1), "token": 2 ** 32 // (page - 1), "head": 2 ** 32 // (H - 1)}[axis] // 64 * 64 + 64

    def pool(far):
        strides = [page * H * D, H * D, D]
        if far:  # the other axes close together
            strides = {"page": strides, "token": [H * D, step, D], "head": [page * D, D, step]}[axis]
            if axis == "page":
                strides[0] = step
        n = 1 + sum(s * (k - 1) for s, k in zip((*strides, 1), (pages, page, H, D)))
        return torch.zeros((n * dtype.itemsize,), dtype=torch.uint8, device=device).view(dtype).as_strided(
            (pages, page, H, D), (*strides, 1))

    q = torch.randn((B, 1, Hq, D), generator=gen, device=device).to(torch.bfloat16)
    k, v = (torch.randn((B, 1500, H, D), generator=gen, device=device).to(torch.bfloat16) for _ in range(2))
    results = []
    for far in (False, True):
        exps = [torch.zeros((pages, H, page), dtype=torch.uint8, device=device) for _ in range(2)] if held == "e4m3" else ()
        cache = PagedCache(pool(far), pool(False), table, *exps)
        assert cache.unwritable is None
        lengths = write_pages(cache, k, v, new_lengths=[1500, 700])
        results.append([lengths, paged_decode(q, cache, kv_lengths=lengths), *read_pages(cache, kv_lengths=lengths)])
        del cache
    torch.cuda.synchronize()
    for a, b in zip(*results):
        assert torch.equal(a, b)


def test_new_rows_far_apart(device):
    import torch
    from probjax_amd.attention import PagedCache, read_pages, write_pages

    T, H, D, step = 150, 2, 64, 2 ** 24 + 8
    near = torch.randn((1, T, H, D), device=device).to(torch.bfloat16)
    wide = torch.empty(((T - 1) * step + H * D,), dtype=torch.bfloat16, device=device)
    far = wide.as_strided((1, T, H, D), (0, step, D, 1))
    far.copy_(near)
    out = []
    for x in (near, far):
        cache = PagedCache.allocate(1, T, H, D, dtype=torch.float8_e4m3fn, device=device)
        write_pages(cache, x, near)
        out.append(read_pages(cache))
    torch.cuda.synchronize()
    assert torch.equal(out[0][0], out[1][0]) and torch.equal(out[0][1], out[1][1])
