"""CPU: what goes into a paged step beside its notes -- second sequence, context, style -- holds the step's own rows."""
import pytest
import torch


class Embedded(Exception):
    """The call went on to the embeddings, whose kernels this test does not run."""


@pytest.mark.parametrize("style_mode", ["adanorm", "cat"])
@pytest.mark.parametrize("width", [1, 3])
def test_paged_steps_refuse_the_rows_of_whole_sequences(style_mode, width):
    from scoreperformer_amd.models import ScorePerformer
    from scoreperformer_amd.modules.transformer import PagedKVCache, PagedStep
    from scoreperformer_amd.synthetic import model_config
    dec = ScorePerformer.init(model_config("tiny", style_emb_mode=style_mode)).eval().perf_decoder.model
    R, K = 2, len(dec.token_emb.num_tokens)
    cache = PagedKVCache(dec.transformer, num_pages=8, max_requests=R, max_len=30, page_size=8)
    step = PagedStep(cache, torch.zeros(R, width, dtype=torch.int64), torch.ones(R, width, dtype=torch.bool), torch.ones(R, dtype=torch.int32))

    def embeds(*_):
        raise Embedded
    dec.token_emb.register_forward_pre_hook(embeds)

    def call(**rows):
        n = {**dict(x=width, x_extra=width, context=width, style=width), **rows}
        with torch.no_grad():
            dec(torch.zeros(R, n["x"], K, dtype=torch.int64), x_extra=torch.zeros(R, n["x_extra"], K, dtype=torch.int64),
                context=torch.zeros(R, n["context"], dec.context_emb_dim), style_embeddings=torch.zeros(R, n["style"], dec.style_emb_dim), paged=step)

    whole = 12
    for name in ("x", "x_extra", "context", "style"):
        with pytest.raises(ValueError, match=f"{name}.* rows of the paged step"):
            call(**{name: whole})
    with pytest.raises(Embedded):                                  # the step's own rows
        call()
    if style_mode == "adanorm":                                    # one style for all rows of a request, as the adaptive norm takes it
        with pytest.raises(Embedded):
            call(style=1)
    elif width > 1:
        with pytest.raises(ValueError, match="style"):
            call(style=1)
