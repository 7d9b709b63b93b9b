"""GPU: reorder_states and select_states against indexing with torch: bits equal."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _pool(rows, seed, small=False):
    """Tensors of a serving pool: matrix states, conv caches, odd-sized and unaligned ones, bytes."""
    gen = torch.Generator("cuda").manual_seed(seed)
    r = lambda *s: torch.randn(rows, *s, generator=gen, device="cuda")
    pool = [r(2, 16, 32), r(3, 96), r(7), r(5, 3).bfloat16(), (r(11) * 50).to(torch.int8)]
    base = torch.randn(rows * 33 + 1, generator=gen, device="cuda")
    pool.append(base[1:].view(rows, 33))  # 4-byte aligned
    return pool[:2] if small else pool + [r(1 << 14)]


def _want(t, index):
    idx = torch.as_tensor(index, device=t.device).long()
    new = t[idx.clamp(min=0)] if t.shape[0] else t.new_zeros((len(index), *t.shape[1:]))
    new[idx < 0] = 0
    return new


def _indices(rows, seed):
    gen = torch.Generator().manual_seed(seed)
    keep = list(range(rows))
    turn = [(d + 1) % rows for d in range(rows)]
    back = [rows - 1 - d for d in range(rows)]
    fork = [0] * rows
    free = [-1] * rows
    mixed = torch.randint(-1, rows, (rows,), generator=gen).tolist()
    shuffled = torch.randperm(rows, generator=gen).tolist()
    chain = [max(0, d - 1) for d in range(rows)]  # every row's source is itself overwritten
    return [keep, turn, back, fork, free, mixed, shuffled, chain]


@pytest.mark.parametrize("rows", [1, 2, 7, 64, 257, 1000, 4096])
def test_reorder_in_place(rows):
    import burn_gdn2 as bg

    for k, index in enumerate(_indices(rows, rows)):
        pool = _pool(rows, k, small=rows > 1000)
        want = [_want(t, index) for t in pool]
        where = (index, torch.tensor(index), torch.tensor(index, dtype=torch.int32, device="cuda"),
                 torch.tensor(index, device="cuda"))[k % 4]
        assert bg.reorder_states(pool, where) is None
        for t, w in zip(pool, want):
            assert torch.equal(t, w), (k, t.shape)
    assert bg._lib.read_device_errors() == 0


@pytest.mark.parametrize("rows,picked", [(5, 3), (3, 9), (64, 64), (2, 4096), (300, 1), (0, 4), (4, 0)])
def test_select_into_another_pool(rows, picked):
    import burn_gdn2 as bg

    gen = torch.Generator().manual_seed(rows)
    index = torch.randint(-1, rows, (picked,), generator=gen).tolist() if rows else [-1] * picked
    pool = _pool(rows, 3, small=picked > 1000)
    before = [t.clone() for t in pool]
    new = bg.select_states(tuple(pool), index)
    assert isinstance(new, tuple)
    for t, b, n in zip(pool, before, new):
        assert torch.equal(t, b)
        assert n.dtype == t.dtype and torch.equal(n, _want(t, index))


def test_layer_states_serve_on():
    """A batch of running layers: forked, compacted and freed rows go on as sequences of their own would."""
    import burn_gdn2 as bg

    cfg = bg.Gdn2Config(hidden_size=64, num_heads=2, head_dim=32)
    layers = [bg.GatedDeltaNet2.new(cfg, device="cuda", seed=s) for s in (1, 2)]
    gen = torch.Generator("cuda").manual_seed(9)
    x = torch.randn(4, 6, 64, generator=gen, device="cuda")
    step = torch.randn(4, 1, 64, generator=gen, device="cuda")

    def states(rows):
        return [m.forward(x[rows])[1] for m in layers]

    live = states([0, 1, 2, 3])
    # sequence 1 ended: 3 moves into its place; row 3 starts again; 2 is forked from 0
    bg.reorder_states(live, [0, 3, 0, -1])
    want = states([0, 3, 0])
    for m, a, b in zip(layers, live, want):
        ya, _ = m.forward(step, a)
        yb, _ = m.forward(step[:3], b)
        assert torch.allclose(ya[:3], yb, rtol=1e-5, atol=1e-6)
        assert torch.equal(a.recurrent[:3].isfinite(), b.recurrent.isfinite())
    fresh = bg.Gdn2State.zeros("cuda", 1, 2, 32, 32, 64, 64)
    y3, _ = layers[0].forward(step[3:], fresh)
    again = states([0, 1, 2, 3])[0]
    bg.reorder_states(again, [0, 1, 2, -1])
    y, _ = layers[0].forward(step, again)
    assert torch.allclose(y[3:], y3, rtol=1e-5, atol=1e-6)
    grown = bg.select_states(states([0, 1, 2, 3]), [3, 3, -1, 0, 1, 2])
    assert isinstance(grown[0], bg.Gdn2State) and grown[1].recurrent.shape[0] == 6


def test_more_tensors_than_a_launch_takes():
    import burn_gdn2 as bg

    pool = [torch.randn(9, 5 + k, device="cuda") for k in range(40)]
    index = [8, 0, 1, 2, -1, 5, 5, 3, 3]
    want = [_want(t, index) for t in pool]
    bg.reorder_states(pool, index)
    assert all(torch.equal(t, w) for t, w in zip(pool, want))


def test_numbers_outside_the_pool():
    """From the host they are refused; on the device their rows stay, the others move, and the error bit says so."""
    import burn_gdn2 as bg

    t = torch.randn(6, 40, device="cuda")
    for bad in ([0, 1, 2, 3, 4, 6], [0, 1, -2, 3, 4, 5], torch.tensor([9] * 6)):
        with pytest.raises(ValueError, match="row numbers"):
            bg.reorder_states(t, bad)
    for dtype in (torch.int32, torch.int64):
        for wild in (6, -2, 2 ** 31 - 1, -2 ** 31) + ((2 ** 32, 2 ** 40) if dtype == torch.int64 else ()):
            before = t.clone()
            bg.reorder_states(t, torch.tensor([1, wild, 0, 3, -1, wild], dtype=dtype, device="cuda"))
            want = _want(before, [1, 1, 0, 3, -1, 5])
            assert torch.equal(t, want)
            assert bg._lib.read_device_errors() == 2
            new = bg.select_states(t, torch.tensor([wild, 2], dtype=dtype, device="cuda"))
            assert torch.equal(new, _want(t, [-1, 2])) and bg._lib.read_device_errors() == 2
    assert bg._lib.read_device_errors() == 0


def test_refusals():
    import burn_gdn2 as bg

    t = torch.zeros(4, 8, device="cuda")
    for pool, index in ((t, [0, 1, 2]), (t, torch.zeros(4, device="cuda")), (t.t(), [0] * 8), ([t, t[:3]], [0] * 4),
                        ([t, t], [0, 1, 2, 3]), ([t, t.view(-1)[:4]], [0, 1, 2, 3]), (t, [[0, 1, 2, 3]]),
                        (torch.zeros(4097, 1, device="cuda"), [0] * 4097), (t.clone().requires_grad_(True), [0, 1, 2, 3])):
        with pytest.raises(ValueError):
            bg.reorder_states(pool, index)
    with pytest.raises(TypeError):
        bg.reorder_states("pool", [0])
    with pytest.raises(RuntimeError, match="CPU tensor"):
        bg.reorder_states(t.cpu(), [0, 1, 2, 3])
    bg.reorder_states([], [])
    bg.reorder_states(t[:0], [])
    assert bg.select_states([], []) == []


def test_captured_call_follows_the_index():
    import burn_gdn2 as bg

    pool = _pool(12, 5)
    index = torch.arange(12, dtype=torch.int32, device="cuda")
    graph = bg.GraphedCall(lambda i: bg.reorder_states(pool, i), index)
    for seed in range(3):
        new = torch.randint(-1, 12, (12,), generator=torch.Generator().manual_seed(seed))
        want = [_want(t, new.tolist()) for t in pool]
        index.copy_(new.cuda())
        graph.replay()
        assert all(torch.equal(t, w) for t, w in zip(pool, want))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    want = [_want(t, [11 - d for d in range(12)]) for t in pool]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        bg.reorder_states(pool, [11 - d for d in range(12)])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(t, w) for t, w in zip(pool, want))


def test_rows_beyond_32_bit_offsets():
    """A pool of more than 4 GB."""
    import burn_gdn2 as bg

    if torch.cuda.mem_get_info()[0] < 8 << 30:
        pytest.skip("needs 8 GB of free device memory")
    t = torch.zeros(5, 1 << 28, device="cuda")  # 5 GB
    t[4, -3:] = torch.tensor([1.0, 2.0, 3.0], device="cuda")
    t[0, :3] = torch.tensor([4.0, 5.0, 6.0], device="cuda")
    bg.reorder_states(t, [4, 1, 2, 3, 0])
    assert t[0, -3:].tolist() == [1, 2, 3] and t[4, :3].tolist() == [4, 5, 6] and not t[0, :3].any() and not t[1:4].any()
