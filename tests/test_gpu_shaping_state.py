"""The state behind the shaping of logits, through the entry point: windows longer than any history, answers of many steps."""
import pytest

from helpers import make_folder, random_tokens

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(tmp_path_factory):
    import gogguf_b200 as gg
    return gg.load(make_folder(tmp_path_factory.getbasetemp(), "L", "float32", scale=4.0), gg.LoadOptions(dtype="float32", max_tokens=64 * 60)).new_context()


def test_a_window_longer_than_any_history(ctx, monkeypatch):
    """It keeps what prompts and answers hold, not what it is asked for, and draws what a window without an end draws."""
    import gogguf_b200 as gg
    from gogguf_b200.sampling import shaping
    shapes, was = [], shaping.ShapingState.__init__

    def init(self, *a, **kw):
        was(self, *a, **kw)
        shapes.append(tuple(self.hist.shape))

    monkeypatch.setattr(shaping.ShapingState, "__init__", init)
    V = ctx.engine.model.spec.vocab_size
    prompts = [random_tokens(V, n, n) for n in (80, 2)]
    kw = dict(max_tokens=9, stop_token_ids=[], repeat_penalty=1.2, frequency_penalty=2.0, logit_bias={4: 1.0})
    endless = [r.tokens for r in ctx.generate(prompts, gg.GenerateParams(repeat_last_n=-1, **kw))]
    shapes.clear()
    assert [r.tokens for r in ctx.generate(prompts, gg.GenerateParams(repeat_last_n=1_000_000, **kw))] == endless
    assert shapes == [(2, 89)]
    shapes.clear()
    assert [r.tokens for r in ctx.generate(prompts, gg.GenerateParams(repeat_last_n=1_000_000, keep_logits=True, **kw))] == endless
    assert shapes == [(2, 80 + k) for k in range(9)]
