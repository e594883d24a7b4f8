"""The cache and position operators in turn, as a serving loop calls them: a
prompt with rotary positions, whose keys collect their weights; eviction into
spare caches; a drafted tree appended, verified and one of its paths kept; a
decode step that goes on collecting weights; eviction again.  Every step's
result is checked against the definition in float64, fed with what the step was
given on the device; tolerances are those of the operators' own tests.
"""

import math

import numpy as np
import pytest

from oracle import cache_ops as ref
from tests._helpers import to_np
from tests.test_gpu_key_weights import check_weights
from tests.test_gpu_rotary import _close
from tests.test_gpu_tree_attention import _types, check

pytestmark = pytest.mark.gpu


class _Loop:
    """One layer's caches and what the loop does with them."""

    def __init__(self, device, dtype, B, Hq, Hkv, D, room, sections, seed):
        import torch

        self.device, self.dtype, self.room, self.sections = device, dtype, room, sections
        self.B, self.Hq, self.Hkv, self.D = B, Hq, Hkv, D
        self.gen = torch.Generator(device=device).manual_seed(seed)
        self.scale = 1.0 / math.sqrt(D)

    def qkv(self, T):
        import torch

        return [torch.randn((self.B, T, h, self.D), generator=self.gen, device=self.device).to(self.dtype)
                for h in (self.Hq, self.Hkv, self.Hkv)]

    def spare(self):
        """Caches with room, laid out ``[B, H, S, D]``; NaN where nothing was written."""
        import torch

        k, v = (torch.full((self.B, self.Hkv, self.room, self.D), float("nan"), dtype=self.dtype,
                           device=self.device).transpose(1, 2) for _ in range(2))
        return k, v, torch.zeros((self.B, self.Hkv, self.room), device=self.device)

    def turn(self, q, k, positions):
        from probjax_amd.attention import rotary

        y, z = rotary(q, k, positions, sections=self.sections)
        pos = np.broadcast_to(to_np(positions), (self.B,) + tuple(positions.shape[-2:]))
        for x, got in ((q, y), (k, z)):
            want = ref.rotary(to_np(x), pos, self.sections)
            _close(got, x, want, self.dtype, None, self.sections, True, False)
        return y, z

    def evict(self, k, v, w, keep, lengths, sinks, recent):
        from probjax_amd.attention import evict_keys

        kept = evict_keys(k, v, w, keep, kv_lengths=lengths, sinks=sinks, recent=recent, out=self.spare())
        n = to_np(lengths) if lengths is not None else [k.shape[1]] * self.B
        for b in range(self.B):
            for h in range(self.Hkv):
                at = ref.evict(to_np(w[b, h]).astype(np.float32), int(n[b]), keep, sinks, recent)
                assert kept.index[b, h].tolist() == at + [-1] * (keep - len(at))
                for x, y in ((k, kept.k), (v, kept.v)):
                    assert np.array_equal(to_np(y[b, :len(at), h]), to_np(x[b, at, h]))
                assert np.array_equal(to_np(kept.key_weights[b, h, :len(at)]), to_np(w[b, h, at]))
            assert int(kept.kv_lengths[b]) == len(at)
        return kept

    def append(self, cache, new, lengths):
        """``new [B, T, H, D]`` behind every sequence's keys."""
        import torch

        T = new.shape[1]
        at = lengths.long()[:, None] + torch.arange(T, device=self.device)
        cache[torch.arange(self.B, device=self.device)[:, None], at] = new


def _np(*xs):
    return [np.nan_to_num(to_np(x).astype(np.float64)) for x in xs]


@pytest.mark.parametrize("name,B,Hq,Hkv,D,prompt,keep,T,sections", [
    ("bf16", 2, 8, 2, 64, 150, 96, 12, (16, 24, 24)),
    ("f16", 1, 4, 4, 128, 260, 130, 33, (128,)),
    ("f32", 2, 4, 1, 64, 97, 40, 5, (64,)),
    ("bf16", 2, 4, 2, 80, 70, 33, 20, (26, 26, 26)),
])
def test_a_serving_loop(device, name, B, Hq, Hkv, D, prompt, keep, T, sections):
    import torch
    from probjax_amd import masks
    from probjax_amd.attention import attention_with_key_weights, tree_attention

    dtype, A = _types()[name], len(sections)
    loop = _Loop(device, dtype, B, Hq, Hkv, D, keep + T + 2, sections, 3)
    # the prompt
    q, k, v = loop.qkv(prompt)
    positions = torch.arange(prompt, device=device)[:, None] // torch.tensor([1, 3, 7][:A], device=device)
    q, k = loop.turn(q, k, positions)
    print("prompt", flush=True)
    out, w, lse = attention_with_key_weights(q, k, v, mask=masks.CausalMask(), return_lse=True)
    zero = np.zeros((B, Hkv, prompt))
    see = np.broadcast_to(np.tri(prompt, dtype=bool), (B, prompt, prompt))
    want = ref.key_weight_attention(*_np(q, k, v), zero, see, loop.scale)
    check(out, lse, want, dtype, D, prompt)
    check_weights(w, want, zero, D, prompt, prompt * Hq // Hkv)
    print("evict", flush=True)
    kept = loop.evict(k, v, w, keep, None, 2, 8)
    L = kept.kv_lengths
    # a drafted tree, some of its tokens missing in the last sequence
    rng = np.random.default_rng(T)
    parents = np.stack([[t - 1 - int(rng.integers(0, min(t + 1, 3))) for t in range(T)] for _ in range(B)])
    parents[-1, T - 2:] = -2
    depth = np.zeros((B, T), np.int64)
    for b in range(B):
        for t in range(T):
            depth[b, t] = depth[b, parents[b, t]] + 1 if parents[b, t] >= 0 else 0
    q, k, v = loop.qkv(T)
    positions = torch.from_numpy(prompt + depth).to(device)[..., None].expand(B, T, A)
    q, k = loop.turn(q, k, positions)
    loop.append(kept.k, k, L)
    loop.append(kept.v, v, L)
    print("tree", flush=True)
    out, lse = tree_attention(q, kept.k, kept.v, parents=parents, kv_lengths=L, return_lse=True)
    sees, token = zip(*(ref.tree_sees(p) for p in parents))
    want = ref.tree_attention(*_np(q, kept.k, kept.v), L.tolist(), sees, token, loop.scale)
    check(out, lse, want, dtype, D, keep + T)
    # a path is kept: its keys move behind the prefix, whose first they follow
    path = [0]
    while len(path) < 3:
        nxt = [t for t in range(path[-1] + 1, T) if parents[0, t] == path[-1]]
        if not nxt:
            break
        path.append(nxt[0])
    for cache, new in ((kept.k, k), (kept.v, v)):
        loop.append(cache, new[:, path], L)
    L = L + len(path)
    # a decode step, whose keys' weights go on from those that eviction kept
    q, k, v = loop.qkv(1)
    positions = torch.full((B, 1, A), prompt + len(path), device=device)
    q, k = loop.turn(q, k, positions)
    loop.append(kept.k, k, L)
    loop.append(kept.v, v, L)
    L = L + 1
    print("decode", flush=True)
    out, w, lse = attention_with_key_weights(q, kept.k, kept.v, kept.key_weights, mask=masks.KVLenMask(L),
                                             return_lse=True)
    see = np.arange(loop.room)[None, None, :] < to_np(L)[:, None, None]
    base = to_np(kept.key_weights).astype(np.float64)
    want = ref.key_weight_attention(*_np(q, kept.k, kept.v), base, see, loop.scale)
    check(out, lse, want, dtype, D, loop.room)
    check_weights(w, want, base, D, loop.room, Hq // Hkv)
    print("evict again", flush=True)
    loop.evict(kept.k, kept.v, w, keep // 2, L, 1, len(path) + 1)


def test_a_captured_step_with_gradients_elsewhere(device):
    """Rotary positions, a drafted tree, a decode step and eviction as one
    captured graph, replayed on new inputs between eager steps, a rotary gradient
    among them."""
    import torch
    from probjax_amd import masks
    from probjax_amd.attention import attention_with_key_weights, evict_keys, rotary, tree_attention

    B, S, T, Hq, Hkv, D, keep = 2, 400, 6, 8, 2, 64, 100
    gen = torch.Generator(device=device).manual_seed(1)

    def new(*shape):
        return torch.randn(shape, generator=gen, device=device).to(torch.bfloat16)

    q, k, v = new(B, T, Hq, D), new(B, S, Hkv, D), new(B, S, Hkv, D)
    w = torch.rand((B, Hkv, S), generator=gen, device=device)
    L = torch.tensor([300, 150], dtype=torch.int32, device=device)
    pos = torch.arange(T, device=device)
    parents = torch.tensor([-1, 0, 0, 1, 1, 2], dtype=torch.int32, device=device)

    def step():
        y = rotary(q, None, pos)
        tree = tree_attention(y, k, v, parents=parents, kv_lengths=L)
        out, sums = attention_with_key_weights(y[:, :1], k, v, w, mask=masks.KVLenMask(L))
        return (tree, out, sums, *evict_keys(k, v, sums, keep, kv_lengths=L, sinks=4, recent=10))

    side = torch.cuda.Stream(device)
    side.wait_stream(torch.cuda.current_stream(device))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(device).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    x = new(B, T, Hq, D).requires_grad_()
    for i in range(4):
        q.copy_(new(B, T, Hq, D))
        k.copy_(new(B, S, Hkv, D))
        w.copy_(torch.rand(w.shape, generator=gen, device=device))
        L.copy_(torch.tensor([300 - 70 * i, 90 + 20 * i], device=device))
        pos.add_(17)
        graph.replay()
        (g,) = torch.autograd.grad(rotary(x, None, pos).float().sum(), x)
        torch.cuda.synchronize()
        for a, b in zip(got, step()):
            assert torch.equal(a, b), i
        ones = torch.ones_like(x)
        assert torch.equal(g, rotary(ones, None, -pos))
