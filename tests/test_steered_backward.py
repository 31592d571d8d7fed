"""What viola_route_steered_backward refuses before any launch."""


def test_rejected_calls_launch_nothing():
    from viola_amd import _lib
    lib, P = _lib.library(), 0x10000

    def call(**changed):
        a = dict(logits=P, pitch=64, dtype=0, tokens=8, experts=64, top_k=4, score=1, normalize=1, scale=1.0, sequence=8, chosen=P, cost=P, stats=P, dgates=P, dloss=P, dlogits=P, stream=None)
        return lib.viola_route_steered_backward(*{**a, **changed}.values())

    for bad in (dict(dtype=3), dict(score=2), dict(tokens=-8), dict(sequence=3), dict(pitch=63), dict(chosen=None), dict(cost=None), dict(stats=None), dict(stats=P + 4), dict(cost=P + 4),
                dict(dlogits=None), dict(logits=None), dict(top_k=0)):
        assert call(**bad) == -1, bad
    assert call(experts=2048, pitch=2048) == -2 and call(top_k=33) == -2
    assert call(tokens=0, sequence=1) == 0
