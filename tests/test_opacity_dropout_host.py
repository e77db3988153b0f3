"""The training step's opacity dropout on the CPU: which offsets it draws under."""

from types import SimpleNamespace


def test_every_step_and_rank_has_its_own_offset(monkeypatch):
    """Ranks of one step and steps of one rank never draw alike, and the
    gradient goes back through the draw of its own step and rank."""
    import dropout
    from data_parallel import DataParallelTrainer

    seen = {}
    now = []

    def apply(x, p, seed, offset, out=None):
        assert (x, p, seed, out) == ("opacity", 0.25, 9, "dropped")
        seen.setdefault(offset, []).append(tuple(now))

    monkeypatch.setattr(dropout, "apply", apply)
    trainer = object.__new__(DataParallelTrainer)
    trainer.opacity_dropout, trainer.dropout_seed = 0.25, 9
    for world in (1, 2, 8):
        seen.clear()
        for t in range(5):
            for rank in range(world):
                now[:] = t, rank
                trainer.adam = SimpleNamespace(t=t, world=world, rank=rank)
                trainer._drop("opacity", "dropped")  # the forward pass
                trainer._drop("opacity", "dropped")  # the gradient
        assert len(seen) == 5 * world
        assert all(len(draws) == 2 and draws[0] == draws[1] for draws in seen.values())
