"""GPU parity of fused attention (forward, gradients, lse) with its definition in 64 bits, element by element and within the
bounds that ``oracle.attention`` derives from the roundings the kernels are allowed; its masks, layouts, streams and captures."""
from __future__ import annotations

import itertools

import pytest
import torch

from oracle import attention as OA

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
DEV = "cuda"


def _rand(seed, *shape, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, device=DEV, generator=g) * std).to(BF16)


def _within(name, got, pair):
    want, bound = pair
    got = got.double()
    assert got.shape == want.shape, name
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)), f"{name}: not finite in other places"
    off = torch.where(torch.isfinite(want), (got - want).abs() - bound, torch.zeros_like(want))
    worst = off.argmax()
    assert float(off.flatten()[worst]) <= 1e-30, (
        f"{name}: {float(got.flatten()[worst])} for {float(want.flatten()[worst])} +- {float(bound.flatten()[worst])} at {int(worst)}; "
        f"{int((off > 1e-30).sum())} of {off.numel()} outside")


def _tensors(B, Lq, Lk, H, Hk, D, seed=0, std=1.0):
    return (_rand(seed, B, Lq, H, D, std=std), _rand(seed + 1, B, Lk, Hk, D, std=std), _rand(seed + 2, B, Lk, Hk, D),
            _rand(seed + 3, B, Lq, H, D, std=0.1))


def _check(q, k, v, g, lengths=None, causal=False, scale=None):
    from anima_trainer_sm120_b200 import _lib
    from anima_trainer_sm120_b200.attention_kernel import fused_attention
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out, lse = fused_attention(*leaves, kv_lengths=lengths, causal=causal, scale=scale, return_lse=True)
    grads = torch.autograd.grad(out, leaves, g)
    with torch.no_grad():
        alone = fused_attention(q, k, v, kv_lengths=lengths, causal=causal, scale=scale)
    torch.cuda.synchronize()
    _lib.check_status_word(torch.device(DEV, torch.cuda.current_device()))
    assert torch.equal(alone, out.detach())
    want = OA.attention(q, k, v, lengths=lengths, causal=causal, scale=scale, dout=g)
    _within("out", out.detach(), want["out"])
    _within("lse", lse, want["lse"])
    for n, t in zip(("dq", "dk", "dv"), grads):
        assert t.dtype == BF16 and t.is_contiguous()
        _within(n, t, want[n])
    return out.detach(), lse, grads


# lengths around the tiles' edges (64, 128, 256), one token, more queries than keys and the reverse, shared key heads
SIZES = [(1, 1, 1, 1, 1, 64), (1, 1, 1, 2, 1, 128), (2, 1, 300, 8, 2, 128), (1, 1, 2049, 4, 4, 64), (2, 64, 64, 4, 4, 64),
         (1, 127, 129, 2, 2, 128), (1, 128, 128, 1, 1, 128), (2, 129, 127, 4, 2, 64), (1, 255, 257, 2, 1, 128),
         (1, 256, 256, 2, 2, 64), (1, 257, 640, 3, 3, 128), (3, 33, 77, 6, 2, 128), (1, 640, 64, 2, 2, 128), (2, 385, 385, 4, 1, 64),
         (1, 1000, 1000, 2, 2, 128), (1, 2, 5000, 2, 1, 128)]


@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("causal", [False, True])
def test_every_size(size, causal):
    _check(*_tensors(*size, seed=sum(size)), causal=causal)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_lengths_leave_samples_and_rows_empty_and_hide_what_lies_behind(D, causal):
    """Lengths of 0, 1, inside a tile, at its edge and all; K and V hold NaN and infinities behind them."""
    n = torch.tensor([0, 1, 127, 128, 130, 300], device=DEV, dtype=torch.int32)
    q, k, v, g = _tensors(6, 200, 300, 4, 2, D, seed=7)
    behind = torch.arange(300, device=DEV)[None] >= n[:, None]
    for t, bad in ((k, float("nan")), (v, float("inf"))):
        t[behind] = bad
        t[behind & (torch.arange(300, device=DEV) % 3 == 0)] = float("nan")
    out, lse, (dq, dk, dv) = _check(q, k, v, g, lengths=n, causal=causal)
    assert not out[0].any() and bool((lse[0] == -float("inf")).all()) and not dq[0].any()
    assert not dk.permute(0, 1, 2, 3)[behind].any() and not dv[behind].any()


def test_causal_with_more_queries_than_keys_leaves_the_first_rows_empty():
    q, k, v, g = _tensors(1, 300, 140, 2, 2, 128, seed=9)
    out, lse, (dq, _, _) = _check(q, k, v, g, causal=True)
    assert not out[:, :160].any() and not dq[:, :160].any() and bool((lse[:, :, :160] == -float("inf")).all())


@pytest.mark.parametrize("D", [64, 128])
def test_what_empty_rows_hold_has_no_part_in_anything(D):
    """Causal, more queries than keys, NaN in q and in the incoming gradient of the queries that see no key."""
    from anima_trainer_sm120_b200.attention_kernel import fused_attention
    q, k, v, g = _tensors(1, 500, 190, 4, 2, D, seed=15)
    results = []
    for bad in (0.0, float("nan")):
        q[:, :310] = bad
        g[:, :310] = bad
        leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
        out = fused_attention(*leaves, causal=True)
        results.append([out.detach(), *torch.autograd.grad(out, leaves, g)])
    assert all(bool(torch.isfinite(b).all()) and torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("lengths", [[2 ** 31 - 1, -5], [400, 0]])
def test_lengths_outside_the_keys_are_clamped(lengths):
    q, k, v, g = _tensors(2, 70, 100, 2, 2, 64, seed=3)
    n = torch.tensor(lengths, device=DEV, dtype=torch.int64 if lengths[0] == 400 else torch.int32)
    _check(q, k, v, g, lengths=n.clamp(0, 100).int())
    from anima_trainer_sm120_b200.attention_kernel import fused_attention
    assert torch.equal(fused_attention(q, k, v, kv_lengths=n), fused_attention(q, k, v, kv_lengths=n.clamp(0, 100)))


@pytest.mark.parametrize("std,scale", [(6.0, None), (1.0, 3.0), (1.0, 1e-6)])
def test_large_and_small_scores(std, scale):
    """One key takes nearly the whole row; rows whose maximum grows from tile to tile; all keys the same."""
    q, k, v, g = _tensors(1, 300, 700, 2, 2, 128, seed=11, std=std)
    k = (k.float() * torch.linspace(0.2, 1.5, 700, device=DEV)[None, :, None, None]).to(BF16)
    _check(q, k, v, g, scale=scale)


def test_scores_that_all_lie_far_below_zero():
    q, k, v, g = _tensors(1, 130, 260, 1, 1, 64, seed=12)
    q, k = q.abs(), -k.abs() * 8
    _check(q, k, v, g, scale=2.0)


def _layouts():
    """Names and functions (B, L, H, D, seed) -> tensor of other strides or alignment."""
    def heads_first(B, L, H, D, s):
        return _rand(s, B, H, L, D).transpose(1, 2)

    def packed(B, L, H, D, s):
        return _rand(s, B, L, H + 3, D)[:, :, 2:2 + H]

    def padded(B, L, H, D, s):
        return _rand(s, B, L + 5, H, D + 8)[:, 3:3 + L, :, :D]

    def odd_pitch(B, L, H, D, s):               # strides no multiple of 16 bytes: copied
        return _rand(s, B, L, H, D + 1)[..., :D]

    def off_by_one(B, L, H, D, s):              # address no multiple of 16 bytes: copied
        return _rand(s, B * L * H * D + 1)[1:].view(B, L, H, D)

    def dim_first(B, L, H, D, s):
        return _rand(s, D, B, L, H).permute(1, 2, 3, 0)

    def expanded(B, L, H, D, s):
        return _rand(s, B, L, 1, D).expand(B, L, H, D)

    return [heads_first, packed, padded, odd_pitch, off_by_one, dim_first, expanded]


@pytest.mark.parametrize("layout", _layouts(), ids=lambda f: f.__name__)
def test_strides_and_alignment(layout):
    B, L, H, D = 2, 150, 4, 64
    q, k, v, g = (layout(B, L, H, D, s) for s in range(20, 24))
    from anima_trainer_sm120_b200.attention_kernel import fused_attention

    def go(*ts):
        leaves = [t.detach().requires_grad_(True) for t in ts[:3]]
        out = fused_attention(*leaves)
        return (out.detach(), *torch.autograd.grad(out, leaves, ts[3]))

    for a, b in zip(go(q, k, v, g), go(*(t.clone(memory_format=torch.contiguous_format) for t in (q, k, v, g)))):
        assert torch.equal(a, b)
    _check(q, k, v, g)


def test_one_query_token_with_groups_of_heads_and_any_stride():
    for B, Lk, H, Hk, D in [(3, 5000, 16, 4, 128), (2, 700, 16, 1, 64), (1, 130, 6, 3, 128)]:
        q = _rand(1, B, H, 1, D).transpose(1, 2)
        n = torch.tensor([Lk, 1, Lk // 2][:B], device=DEV, dtype=torch.int32)
        _check(q, _rand(2, B, Lk, Hk, D), _rand(3, B, Lk, Hk, D), _rand(4, B, 1, H, D), lengths=n)
        _check(q, _rand(2, B, Lk, Hk, D), _rand(3, B, Lk, Hk, D), _rand(4, B, 1, H, D), causal=True)


def test_gradients_of_differences():
    """The gradients against the change of the (64-bit) loss that a small step along a random direction makes: what the
    kernel calls the gradient is the derivative of what it calls the output, and not only the oracle's formula."""
    from anima_trainer_sm120_b200.attention_kernel import fused_attention
    q, k, v, g = _tensors(1, 70, 200, 2, 1, 64, seed=31)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(fused_attention(*leaves), leaves, g)
    want = OA.attention(q, k, v, dout=g)
    for i, name in enumerate(("dq", "dk", "dv")):
        d = torch.randn(leaves[i].shape, device=DEV, dtype=torch.float64, generator=torch.Generator(DEV).manual_seed(i))
        eps = 1e-4
        ends = []
        for sign in (1, -1):
            ts = [t.double() for t in (q, k, v)]
            ts[i] = ts[i] + sign * eps * d
            ends.append((OA.attention(*ts)["out"][0] * g.double()).sum())
        slope = (ends[0] - ends[1]) / (2 * eps)
        bound = (want[name][1] * d.abs()).sum() + 1e-5 * (want[name][0] * d).abs().sum()     # eps^2 terms of the difference
        assert float(((grads[i].double() * d).sum() - slope).abs()) <= float(bound)


def test_every_subset_of_gradients_gives_the_same_bits():
    from anima_trainer_sm120_b200.attention_kernel import fused_attention
    q, k, v, g = _tensors(2, 200, 150, 4, 2, 128, seed=41)

    def go(subset):
        leaves = [t.clone().requires_grad_(i in subset) for i, t in enumerate((q, k, v))]
        out = fused_attention(*leaves)
        if subset:
            out.backward(g)
        return out.detach(), [t.grad for t in leaves]

    out, grads = go({0, 1, 2})
    for r in range(3):
        for subset in itertools.combinations(range(3), r):
            o, some = go(set(subset))
            assert torch.equal(o, out)
            for i, (a, b) in enumerate(zip(some, grads)):
                assert (a is None) == (i not in subset) and (a is None or torch.equal(a, b))
    again = go({0, 1, 2})[1]
    assert all(torch.equal(a, b) for a, b in zip(again, grads))          # deterministic


def test_one_tensor_as_query_key_and_value():
    from anima_trainer_sm120_b200.attention_kernel import fused_attention
    x = _rand(51, 1, 140, 2, 64).requires_grad_(True)
    g = _rand(52, 1, 140, 2, 64)
    fused_attention(x, x, x).backward(g)
    want = OA.attention(x.detach(), x.detach(), x.detach(), dout=g)
    value = sum(want[n][0] for n in ("dq", "dk", "dv"))
    _within("dx", x.grad, (value, sum(want[n][1] for n in ("dq", "dk", "dv")) * (1 + OA.BF16_HALF) + 2 * OA.BF16_HALF * (
        value.abs() + sum(want[n][0].abs() for n in ("dq", "dk", "dv")))))


def test_empty_tensors():
    from anima_trainer_sm120_b200.attention_kernel import fused_attention
    for B, Lq, Lk in [(0, 5, 5), (2, 0, 5), (2, 5, 0), (0, 0, 0)]:
        ts = [_rand(i, B, L, 2, 64).requires_grad_(True) for i, L in enumerate((Lq, Lk, Lk))]
        out, lse = fused_attention(*ts, return_lse=True)
        assert out.shape == (B, Lq, 2, 64) and not out.any() and bool((lse == -float("inf")).all())
        grads = torch.autograd.grad(out, ts, torch.ones_like(out))
        assert all(a.shape == b.shape and not a.any() for a, b in zip(grads, ts))


def test_refusals():
    from anima_trainer_sm120_b200.attention_kernel import fused_attention
    q, k, v, _ = _tensors(1, 8, 8, 4, 2, 64)
    with pytest.raises(TypeError):
        fused_attention(q.float(), k, v)
    with pytest.raises(TypeError):
        fused_attention(q, k, v.half())
    with pytest.raises(ValueError):
        fused_attention(q[0], k[0], v[0])
    with pytest.raises(ValueError):
        fused_attention(q, k, v[:, :4])
    with pytest.raises(ValueError):
        fused_attention(q[:, :, :3], k, v)                              # 3 heads on 2 key heads
    with pytest.raises(NotImplementedError):
        fused_attention(q[..., :32], k[..., :32], v[..., :32])
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        with pytest.raises(ValueError):
            fused_attention(q, k, v, scale=scale)
    with pytest.raises(ValueError):
        fused_attention(q, k, v, kv_lengths=torch.tensor([8, 8], device=DEV))
    with pytest.raises(TypeError):
        fused_attention(q, k, v, kv_lengths=torch.tensor([8.0], device=DEV))
    with pytest.raises(RuntimeError):
        fused_attention(q, k, v, kv_lengths=torch.tensor([8]))
    with pytest.raises(RuntimeError):
        fused_attention(q.cpu(), k.cpu(), v.cpu())
    x = q.clone().requires_grad_(True)
    with pytest.raises(NotImplementedError):
        torch.autograd.grad(fused_attention(x, k, v).sum(), x, create_graph=True)
    n = torch.tensor([8], device=DEV, dtype=torch.int32)
    out = fused_attention(x, k, v, kv_lengths=n)
    n.fill_(3)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()
    out = fused_attention(x, k, v)
    out.mul_(2)                                                          # the output is read by backward
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()


def test_another_stream_and_two_calls_at_once():
    from anima_trainer_sm120_b200.attention_kernel import fused_attention
    a, b = _tensors(1, 300, 1400, 4, 2, 128, seed=61), _tensors(2, 129, 2000, 4, 4, 64, seed=65)

    def go(ts):
        leaves = [t.detach().requires_grad_(True) for t in ts[:3]]
        out = fused_attention(*leaves, causal=True)
        return (out.detach(), *torch.autograd.grad(out, leaves, ts[3]))

    want = [go(a), go(b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [None, None]
    for _ in range(3):
        for i, (s, ts) in enumerate(zip(streams, (a, b))):
            with torch.cuda.stream(s):
                got[i] = go(ts)
    torch.cuda.synchronize()
    for w, o in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(w, o))


def test_first_call_of_a_new_thread():
    """A thread without a current context: the caller's own, and autograd's worker."""
    import threading
    from anima_trainer_sm120_b200.attention_kernel import fused_attention
    q, k, v, g = _tensors(1, 40, 60, 2, 2, 64, seed=5)
    found = []

    def go():
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = fused_attention(*leaves)
        found.append([out.detach(), *torch.autograd.grad(out, leaves, g)])

    for _ in range(2):
        t = threading.Thread(target=go)
        t.start()
        t.join()
    go()
    torch.cuda.synchronize()
    assert len(found) == 3 and all(torch.equal(a, b) for f in found[:2] for a, b in zip(f, found[2]))


def test_captured_and_replayed_with_other_inputs():
    """Forward and backward in one graph, a second graph beside it, and an eager pass between their replays."""
    from anima_trainer_sm120_b200.attention_kernel import fused_attention
    sizes = [(2, 200, 1300, 4, 2, 128), (1, 1, 3000, 4, 2, 64)]
    lengths = torch.tensor([1300, 700], device=DEV, dtype=torch.int32)

    def go(ts, n):
        out = fused_attention(*ts[:3], kv_lengths=n)
        return (out, *torch.autograd.grad(out, ts[:3], ts[3]))

    kept = []
    for i, size in enumerate(sizes):
        ts = [t.clone() for t in _tensors(*size, seed=70 + i)]
        for t in ts[:3]:
            t.requires_grad_(True)
        n = lengths[:size[0]].clone()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            go(ts, n)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = go(ts, n)
        kept.append((graph, ts, n, outs, size))
    for turn in range(2):
        for i, (graph, ts, n, outs, size) in enumerate(kept):
            new = _tensors(*size, seed=90 + 10 * turn + i)
            with torch.no_grad():
                for t, x in zip(ts, new):
                    t.copy_(x)
                n.sub_(50)
        for graph, *_ in kept:
            graph.replay()
        for graph, ts, n, outs, size in kept:
            fresh = [t.detach().clone().requires_grad_(j < 3) for j, t in enumerate(ts)]
            for a, b in zip(outs, go(fresh, n)):
                assert torch.equal(a.detach(), b.detach())


def test_offsets_beyond_32_bits():
    """Keys and values as one half of a cache whose token pitch puts the last ones behind 2^32 elements."""
    from anima_trainer_sm120_b200.attention_kernel import fused_attention
    pitch, L = 1 << 20, 4200
    free = torch.cuda.mem_get_info()[0]
    if free < 3 * pitch * L:
        pytest.skip("not enough free memory")
    store = torch.empty(pitch * L, device=DEV, dtype=BF16)
    k = store.as_strided((1, L, 2, 64), (pitch * L, pitch, 64, 1))
    v = store.as_strided((1, L, 2, 64), (pitch * L, pitch, 64, 1), 4096)
    small = [_rand(i, 1, L, 2, 64) for i in (81, 82)]
    k.copy_(small[0])
    v.copy_(small[1])
    q = _rand(83, 1, 40, 2, 64)
    assert torch.equal(fused_attention(q, k, v), fused_attention(q, *small))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_more_tiles_than_fit_at_once(D, causal):
    """Two CTAs a SM take all tiles in turn: long, short and empty ones one after the other."""
    n = torch.tensor([0, 641, 1, 0, 0, 320, 63, 65, 0], device=DEV, dtype=torch.int32)
    q, k, v, g = _tensors(9, 641, 641, 16, 8, D, seed=81)
    for b, m in enumerate(n.tolist()):
        k[b, m:], v[b, m:] = float("nan"), float("inf")
    _check(q, k, v, g, lengths=n, causal=causal)


@pytest.mark.parametrize("causal", [False, True])
def test_gradients_of_many_heads_are_those_of_fewer_heads(causal):
    """The backward pass goes through 130 heads of 4096 tokens in uneven parts, through 26 at once."""
    from anima_trainer_sm120_b200.attention_kernel import fused_attention
    q, k, v, g = _tensors(1, 4096, 4096, 130, 130, 64, seed=61)

    def go(a, b):
        leaves = [t[:, :, a:b].detach().requires_grad_(True) for t in (q, k, v)]
        return torch.autograd.grad(fused_attention(*leaves, causal=causal), leaves, g[:, :, a:b])

    whole = go(0, 130)
    for a in range(0, 130, 26):
        for x, y in zip(whole, go(a, a + 26)):
            assert torch.equal(x[:, :, a:a + 26], y)
    _check(q[:, :1000, 129:], k[:, :, 129:], v[:, :, 129:], g[:, :1000, 129:], causal=causal)


def test_causal_heads_in_several_blocks():
    """The tiles of several hundred heads are taken in turn; 656 heads are more than one such block, and not a whole number."""
    n = torch.tensor([130 - i for i in range(41)], device=DEV, dtype=torch.int32)
    _check(*_tensors(41, 130, 130, 16, 16, 64, seed=91), lengths=n, causal=True)
    _check(*_tensors(41, 130, 259, 16, 8, 64, seed=92), causal=True)


@pytest.mark.parametrize("causal", [False, True])
def test_gradients_of_a_key_head_that_serves_very_many_pairs(causal):
    """16 x 11603 x 11603 pairs to a key head: dS is not stored. Element by element against the 64-bit definition, head by head."""
    from anima_trainer_sm120_b200.attention_kernel import fused_attention
    H, L, D = 16, 11603, 64
    q, k, v, g = _tensors(2, L, L, H, 1, D, seed=71)
    n = torch.tensor([L, 6001], device=DEV, dtype=torch.int32)
    k[1, 6001:], v[1, 6001:] = float("nan"), float("inf")
    leaves = [t.requires_grad_(True) for t in (q, k, v)]
    dq, dk, dv = torch.autograd.grad(fused_attention(*leaves, kv_lengths=n, causal=causal), leaves, g)
    for b in range(2):
        sums = {}
        for h in range(H):
            want = OA.attention(q[b:b + 1, :, h:h + 1].detach(), k[b:b + 1].detach(), v[b:b + 1].detach(), lengths=n[b:b + 1],
                                causal=causal, dout=g[b:b + 1, :, h:h + 1])
            _within("dq", dq[b:b + 1, :, h:h + 1], want["dq"])
            for name in ("dk", "dv"):
                value, bound = want[name]
                sums[name] = (sums[name][0] + value, sums[name][1] + bound) if name in sums else (value, bound)
        # the sum over heads is rounded to bf16 once, by no more than the half steps of all heads that the bounds count
        _within("dk", dk[b:b + 1], sums["dk"])
        _within("dv", dv[b:b + 1], sums["dv"])


def test_under_checkpoint():
    from torch.utils.checkpoint import checkpoint
    from anima_trainer_sm120_b200.attention_kernel import fused_attention
    q, k, v, g = _tensors(2, 100, 300, 4, 4, 64, seed=101)
    results = []
    for wrap in (lambda f, *a: f(*a), lambda f, *a: checkpoint(f, *a, use_reentrant=False)):
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        out = wrap(fused_attention, *leaves)
        out.backward(g)
        results.append([out.detach()] + [t.grad for t in leaves])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_thin_wrappers_give_the_nodes_bits():
    from anima_trainer_sm120_b200 import ops
    from anima_trainer_sm120_b200.attention_kernel import fused_attention
    q, k, v, g = _tensors(2, 130, 260, 4, 2, 128, seed=111)
    n = torch.tensor([260, 99], device=DEV, dtype=torch.int32)
    out, lse = ops.attention_fwd(q, k, v, kv_lengths=n, causal=True, scale=0.1)
    grads = ops.attention_bwd(g, q, k, v, out, lse, kv_lengths=n, causal=True, scale=0.1)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    want, want_lse = fused_attention(*leaves, kv_lengths=n, causal=True, scale=0.1, return_lse=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    assert all(torch.equal(a, b) for a, b in zip(grads, torch.autograd.grad(want, leaves, g)))
    with pytest.raises(ValueError):
        ops.attention_fwd(q, k, v[:, :5])
    with pytest.raises(ValueError):
        ops.attention_fwd(q, k, v, kv_lengths=n.long())
    with pytest.raises(ValueError):
        ops.attention_bwd(g, q, k, v, out, lse[:1])
    with pytest.raises(ValueError):
        ops.attention_fwd(q.transpose(2, 3), k, v)
