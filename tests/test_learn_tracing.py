"""The operators on learned node values inside a traced sampler: they are recorded as calls, and two equal
dropout calls stay two draws."""
import torch


def test_lookup_and_dropout_are_recorded_and_draws_are_not_merged():
    import gsampler_b200 as gs
    from gsampler_b200.jit import passes

    def fn(table, ids):
        x = gs.ops.embedding(table, ids, scale=2.0)
        y = gs.ops.embedding(table, ids, scale=2.0)
        return gs.ops.dropout(x, 0.5) + gs.ops.dropout(x, 0.5) + y

    gm = torch.fx.symbolic_trace(fn)
    count = lambda name: sum(name in str(n.target) for n in gm.graph.nodes)
    assert count("_CAPI_EmbeddingLookup") == 2 and count("_CAPI_DropoutApply") == 2
    gm = passes.eliminate_common_subexpressions(gm)
    gm = passes.eliminate_dead_code(gm)
    assert count("_CAPI_EmbeddingLookup") == 1 and count("_CAPI_DropoutApply") == 2
