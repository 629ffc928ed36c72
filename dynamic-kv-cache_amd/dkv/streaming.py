"""Streaming decoder over the packed cache: frame ingestion and candidate scoring.

The caller side of the packed-KV path, following the reference's StreamingModel
(src/streaming.py:89-237) on a text decoder with synthetic frame embeddings in
place of the vision encoder:

- ingest(): one decoder forward for a text prefix, then one per 64-token frame.
  The cache's width is selected per frame (cache.select(bits, i),
  src/streaming.py:178), and every LlamaAttention packs its K/V and attends
  over the packed history (install_packed_attention). With a budget the cache counts the
  frames' attention and evicts the tokens that got least of it, so a stream has no end.
- generate(): tokens drawn one after the other on a fork from given random numbers, each
  attending to all of the history or to the part of it that scores highest for it.
- generate_batch(): the same for many questions at once, about one stream or several, on branches in
  the shared pages of a PagedCache: a forward of all questions, then one forward a token for all.
- answer(): the reference's 'candidate' protocol (src/streaming.py:209-225).
  For each candidate, a fork of the cache runs question + candidate tokens, and
  the score is the mean log-likelihood of the candidate tokens. answer_labels()
  is the 'label' protocol and prior_scores() the prior of 'candidate_calibrated'.
- answer_batched(): the same scores from one forward of the question on a fork,
  then one forward of all candidates together. The candidates sit back to back
  in one chunk with per-candidate positions and a block-diagonal chunk mask
  (GPUCache.chunk_segments), so the shared history is read once per batch
  instead of once per candidate.

The model is a random-init LlamaForCausalLM. There is no checkpoint, and the
workloads are synthetic; see dkv.workloads.decoder_config.
"""
import contextlib

import torch

from .gpu_cache import GPUCache, install_packed_attention
from .gpu_ops import install_fused_ops, sample
from .paged_cache import PagedCache

# generate_batch() captures more tokens than these: a replayed forward of a token of each sequence takes 1.30 to 1.37 ms and an eager
# one, which waits for the host, 1.6 (32 layers, 1 to 16 questions; at 64 1.81 and 1.66, its launches are sized for any step), a capture 3
# to 8 ms.
GRAPH_TOKENS = 16
MFMA_ROWS = 192  # query rows per frame-chunk attention workgroup (MFMA_ROWS of csrc/dkv_attn_common.h)


def build_decoder(layers=32, hidden=960, heads=15, kv_heads=5, intermediate=2560, vocab=49280,
                  rope_theta=100000.0, max_positions=8192, seed=0, device='cuda', dtype=torch.bfloat16):
    """A random-init Llama text decoder of the given shape, on `device`, in eval mode."""
    from transformers import LlamaConfig, LlamaForCausalLM
    config = LlamaConfig(vocab_size=vocab, hidden_size=hidden, intermediate_size=intermediate,
                         num_hidden_layers=layers, num_attention_heads=heads, num_key_value_heads=kv_heads,
                         head_dim=hidden // heads, hidden_act='silu', rms_norm_eps=1e-5,
                         max_position_embeddings=max_positions, rope_theta=rope_theta,
                         tie_word_embeddings=True, attn_implementation='sdpa')
    with torch.random.fork_rng(devices=[]):
        torch.manual_seed(seed)
        model = LlamaForCausalLM(config)
    return model.to(device=device, dtype=dtype).eval()


class StreamingDecoder:
    """Frame-by-frame ingestion into a GPUCache and candidate scoring (src/streaming.py:89-237)."""

    def __init__(self, model, fused_ops=True, precision='bf16', graphs=False, pipeline=8, group_splits=None):
        self.model = model
        self.text = model.model
        self.config = model.config
        self.precision = precision
        self.graphs = graphs
        self.pipeline = pipeline
        # History splits of the frame-chunk attention in pipelined groups (None: group_split_count())
        self.group_splits = group_splits
        self.ops_state = {'enabled': fused_ops}
        install_fused_ops(self.text, self.ops_state)
        install_packed_attention(model)
        self._cache = None  # reused across requests when graphs=True (a captured graph records its buffers)
        self._spare = None  # the cache that _cache evicts into and back, and that cache's captured forwards
        self._graphs = {}  # chunk length -> captured forward of that length on self._cache
        self._group_graphs = {}  # (chunk length, k) -> captured forwards of k consecutive chunks (pipelined)
        self._qa_graphs = {}  # (chunk length, logits, segments) -> captured forward + lm_head on a fork
        self._qa_seen = set()  # QA shapes already run once eagerly (warms the library paths a capture records)

    @property
    def device(self):
        return self.model.lm_head.weight.device

    def group_split_count(self, chunk):
        """History splits per KV head of the frame-chunk attention while frames are pipelined
        (pipeline > 1). The library's default plan gives one launch the whole GPU (one workgroup
        per CU per split), the shortest latency when it runs alone. In a pipelined group several
        frames' launches run at once and the GPU is throughput-bound, so each takes a quarter of
        that: fewer workgroups, each over more units, pay the per-workgroup prologue, merge and
        partial stores fewer times. 96 frames + 4 candidates (5 KV heads, 256 CUs): 1079 frames/s
        at the default 51-split cap, 1134-1139 at 12 splits, 1132-1134 at 16, 1111-1121 at 24,
        1106-1108 at 8; frames one at a time are fastest at the default (586 vs 528 at 12).
        With the later, faster attention kernel 8 to 24 splits all gave 1122-1141 frames/s."""
        if self.group_splits is not None:
            return self.group_splits
        c = self.config
        rows = c.num_attention_heads // c.num_key_value_heads * chunk
        row_groups = -(-rows // MFMA_ROWS)
        cus = torch.cuda.get_device_properties(self.device).multi_processor_count
        return max(1, cus // (c.num_key_value_heads * row_groups) // 4)

    def create_cache(self, max_tokens, **kw):
        c = self.config
        return GPUCache(None, layers=c.num_hidden_layers, heads=c.num_key_value_heads, dim=c.head_dim,
                        dtype=self.model.dtype, max_tokens=max_tokens, precision=self.precision,
                        device=self.device, **kw)

    def create_paged_cache(self, max_tokens, **kw):
        """A PagedCache of the decoder's shape, which adopts the histories that ingest() returned."""
        c = self.config
        return PagedCache(c.num_hidden_layers, c.num_key_value_heads, c.num_attention_heads, max_tokens=max_tokens,
                          dim=c.head_dim, precision=self.precision, device=self.device, **kw)

    @staticmethod
    def _position(cache, past=None):
        """Position of the token after `past` held ones (default: all): evicted tokens keep theirs."""
        return (cache.get_seq_length() if past is None else past) + getattr(cache, 'dropped', 0)

    @torch.inference_mode()
    def forward(self, cache, ids=None, embeddings=None, positions=None, logits=0):
        """One decoder forward of a chunk. Returns fp32 logits of the last `logits` positions.

        With graphs=True a chunk may run here once and as graph replays later, so its attention runs
        the kernels that replays run (GPUCache.as_replayed): the outputs are the same bits either way.
        """
        if embeddings is None:
            embeddings = self.text.get_input_embeddings()(ids.to(self.device))
        n = embeddings.shape[1]
        if positions is None:
            past = self._position(cache)
            positions = torch.arange(past, past + n, device=self.device)
        before, cache.as_replayed = getattr(cache, 'as_replayed', False), True
        try:
            out = self.text(inputs_embeds=embeddings, past_key_values=cache, use_cache=True,
                            position_ids=positions[None], attention_mask=None, return_dict=True)
        finally:
            cache.as_replayed = before
        if not logits:
            return None
        return self.model.lm_head(out.last_hidden_state[:, -int(logits):]).float()

    @torch.inference_mode()
    def ingest(self, prefix_ids, frames, bits, cache=None, qa_reserve=256, budget=None):
        """Prefix at 16 bits, then each frame embedding [1, T, hidden] at its width (src/streaming.py:168-187).

        With graphs=True the frames after the first run as replays of one captured HIP graph of the
        whole decoder forward (the cache's launches read their step parameters from the device), on
        a cache the decoder keeps and resets between requests. With pipeline=k > 1 as well, k
        consecutive frames replay one graph of their k forwards in which frame i + 1's layer l
        waits only for frame i's layer l (the K/V it attends to) and its own layer l - 1: each
        forward runs one layer behind the one before it, on its own stream. The launches and the
        data are those of one frame after the other; the GPU overlaps them. With pipeline > 1 every
        chunk's attention (eager or replayed) runs group_split_count() history splits, so replays
        still equal eager ingestion bit for bit; question and candidate forwards keep the default.

        With a `budget` the history stays within that many tokens. The attention of the prefix and of every
        frame is counted, and before a frame that would pass the budget the tokens of the least attention
        mass are evicted (GPUCache.evict), down to three quarters of the budget (where the prefix fills
        these, of what it leaves) or to what the frame needs. The prefix stays (where the cache held tokens
        before, its first ones instead, as many), and of the frames that the last quarter of the budget takes
        in the newest that leave room for it. A budget that some frame and the prefix use up, or that the
        cache cannot hold, is refused before any forward. The cache that is returned holds the history: with a
        budget it may be another one than the `cache` given, which then holds what it did before the first
        eviction, for its forks too. (With graphs=True the decoder's own cache evicts into another one that
        the decoder keeps, and that one back: as between requests, forks of either end there.)
        """
        if len(frames) != len(bits):
            raise ValueError('one bit width per frame')
        total = prefix_ids.shape[1] + sum(f.shape[1] for f in frames)
        if budget is not None:
            if budget < prefix_ids.shape[1]:
                raise ValueError(f'a budget of {budget} tokens does not hold the prefix of {prefix_ids.shape[1]}')
            self._check_budget(budget, prefix_ids.shape[1], [f.shape[1] for f in frames], cache)
            total = min(total, budget)
        total += qa_reserve
        given = cache
        if cache is None:
            cache = self._reused_cache(total) if self.graphs else self.create_cache(total)
        # pipelined frames share the GPU: their frame-chunk attention takes fewer history splits
        splits = self.group_split_count(max(f.shape[1] for f in frames)) if self.pipeline > 1 and frames else 0
        caches, observing = [cache], getattr(cache, 'observing', False)
        try:
            cache.chunk_splits, cache.observing = splits, observing or budget is not None
            if cache.observing:
                cache.mass()  # (allocated before a capture records it)
            return self._ingest_chunks(caches, given, prefix_ids, frames, bits, budget)
        finally:
            for c in caches:
                c.chunk_splits, c.observing = 0, observing

    @staticmethod
    def _protected(cache, prefix):
        """Tokens at the start of a cache that a budgeted ingest keeps: the segments of the first `prefix` ones."""
        return next((s.end for s in cache.segments if s.end >= prefix), cache.get_seq_length()) if prefix else 0

    @staticmethod
    def _kept(budget, protected, frame):
        """Tokens that an eviction before a frame leaves, of which `protected` stay."""
        keep = budget - budget // 4
        if keep <= protected:
            keep = protected + (budget - protected) * 3 // 4
        return min(keep, budget - frame)

    def _check_budget(self, budget, prefix, frames, cache):
        """Whether every eviction of an ingest leaves what is protected, and something beside it."""
        held, protected = 0, prefix
        if cache is not None:
            if not cache.online:
                raise ValueError('a budget needs an online cache (no plan)')
            held = cache.get_seq_length()
            protected = self._protected(cache, prefix) if held >= prefix else held + prefix
            if cache.capacity < min(budget, held + prefix + sum(frames)):
                raise ValueError(f'a budget of {budget} tokens is more than the {cache.capacity} that the cache holds')
        for n in [prefix] + frames:
            if held + n > budget:
                held = self._kept(budget, protected, n)
                if held <= protected:
                    raise ValueError(f'a budget of {budget} tokens holds no history beside {protected} protected tokens '
                                     f'(the prefix) and {n} new ones')
            held += n

    def _evict_for(self, caches, given, budget, frame, prefix):
        """Room for a frame within the budget: the last of `caches` (those of this ingest) evicts into another of
        them, never the `given` one, or into a new one. That goes to the end of the list and is returned."""
        cache = caches[-1]
        protected = self._protected(cache, prefix)
        keep = self._kept(budget, protected, frame)
        recent, tail = budget // 4, 0
        for seg in reversed(cache.segments):  # whole segments stay: those that leave room for the protected ones
            if tail >= recent:
                break
            if tail + seg.rows > keep - protected:
                recent = tail
                break
            tail += seg.rows
        own = self.graphs and cache is self._cache
        if own:
            if self._spare is None or self._spare[0].capacity < cache.capacity:
                self._spare = (self.create_cache(cache.capacity), {}, {}, {}, set())
            into = self._spare[0]
        else:
            into = next((c for c in caches if c is not cache and c is not given), None)
        new = cache.evict(keep, sinks=prefix, recent=recent, into=into)
        if own:  # captured forwards stay with the cache whose buffers they recorded
            (self._cache, self._graphs, self._group_graphs, self._qa_graphs, self._qa_seen), self._spare = \
                self._spare, (cache, self._graphs, self._group_graphs, self._qa_graphs, self._qa_seen)
        caches[:] = [c for c in caches if c is not new] + [new]
        return new

    @staticmethod
    def _graph_key(cache, *key):
        """Key of a captured forward: one that counts attention or attends sparsely records other launches."""
        if cache.observing:
            key += ('observing',)
        if cache.sparse_blocks:
            key += ('sparse', cache.sparse_blocks)
        return key if len(key) > 1 else key[0]

    @staticmethod
    def _captured(graphs, key, cache):
        """The captured forward under `key`, or None: one whose index or masses the cache no longer holds is dropped,
        to be captured again."""
        fg = graphs.get(key)
        if fg is None:
            return None
        steps = fg['steps'] if isinstance(fg['steps'], list) else [fg['steps']]
        if all(st.replays_on(cache) for st in steps):
            return fg
        torch.cuda.synchronize()  # (it may still run)
        del graphs[key]
        return None

    def _ingest_chunks(self, caches, given, prefix_ids, frames, bits, budget):
        cache = caches[-1]
        n = prefix_ids.shape[1]
        if budget is not None and cache.get_seq_length() + n > budget:
            cache = self._evict_for(caches, given, budget, n, n)
        cache.select(16, -1)
        graphed = self.graphs and cache is self._cache
        # The first request's prefix and first frame run eagerly (they warm up the library paths
        # a capture records); after that every chunk replays the captured forward of its length
        # (captured on first use).
        warm = bool(self._graphs or self._group_graphs)
        if graphed and warm:
            self._graph_chunk(cache, self.text.get_input_embeddings()(prefix_ids.to(self.device)))
        else:
            self.forward(cache, ids=prefix_ids)
        i = 0
        while i < len(frames):
            emb, b = frames[i], bits[i]
            replay = graphed and (i > 0 or warm)
            n, most = emb.shape[1], self.pipeline
            if budget is not None:
                if cache.get_seq_length() + n > budget:
                    cache = self._evict_for(caches, given, budget, n, prefix_ids.shape[1])
                most = min(most, (budget - cache.get_seq_length()) // max(n, 1))
            k = 1
            while k < most and i + k < len(frames) and frames[i + k].shape[1] == n:
                k += 1
            if replay and k > 1:
                self._graph_group(cache, frames[i:i + k], bits[i:i + k], i)
                i += k
                continue
            cache.select(b, i)
            if replay:
                self._graph_chunk(cache, emb)
            else:
                self.forward(cache, embeddings=emb)
            i += 1
        cache.select(16, -1)
        if len(set(cache.seen)) != 1:
            raise RuntimeError('Decoder layers disagree about the cache length')
        return cache

    def _reused_cache(self, total):
        if self._cache is None or self._cache.capacity < total:
            self._cache = self.create_cache(max(total, 8192))
            # a captured graph records the old cache's buffers
            self._graphs, self._group_graphs, self._qa_graphs, self._qa_seen = {}, {}, {}, set()
            self._spare = None
        else:
            self._cache.reset()
        return self._cache

    def _graph_chunk(self, cache, emb):
        """One chunk as a replay of the captured forward of its length (captured on first use)."""
        fg = self._captured(self._graphs, self._graph_key(cache, emb.shape[1]), cache)
        if fg is None:
            self._capture_chunk(cache, emb)
            return
        cache.begin_graph_steps(fg['chunk'], steps=fg['steps'])
        try:
            past = cache.graph_step()
            fg['emb'].copy_(emb)
            torch.add(fg['arange'], self._position(cache, past), out=fg['pos'][0])
            fg['graph'].replay()
        finally:
            cache.end_graph_steps()

    def _capture_chunk(self, cache, emb):
        chunk = emb.shape[1]
        static_emb = emb.clone()
        arange = torch.arange(chunk, device=self.device)
        pos = torch.empty((1, chunk), dtype=torch.long, device=self.device)
        steps = cache.begin_graph_steps(chunk, q_heads=self.config.num_attention_heads)
        try:
            past = cache.graph_step()
            torch.add(arange, self._position(cache, past), out=pos[0])
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                self.text(inputs_embeds=static_emb, past_key_values=cache, use_cache=True, position_ids=pos,
                          attention_mask=None, return_dict=True)
            steps.upload()  # the jobs now carry the K/V addresses recorded in the graph
            graph.replay()
        finally:
            cache.end_graph_steps()
        self._graphs[self._graph_key(cache, chunk)] = dict(chunk=chunk, graph=graph, steps=steps, emb=static_emb, pos=pos, arange=arange)

    def _group_steps(self, cache, chunk, bits, frame, steps):
        """Host bookkeeping of frames frame .. frame + k - 1 (one GraphSteps each, since their
        forwards run at once); returns their first positions and the GraphSteps."""
        past, out = [], []
        for j, st in enumerate(steps):
            cache.select(bits[j], frame + j)
            cache.begin_graph_steps(chunk, q_heads=None if st else self.config.num_attention_heads, steps=st)
            try:
                past.append(self._position(cache, cache.graph_step()))
            finally:
                out.append(cache.end_graph_steps())
        return past, out

    def _graph_group(self, cache, embs, bits, frame):
        """k consecutive frames as one replay of their pipelined forwards (captured on first use)."""
        chunk, k = embs[0].shape[1], len(embs)
        fg = self._captured(self._group_graphs, self._graph_key(cache, chunk, k), cache)
        if fg is None:
            self._capture_group(cache, embs, bits, frame)
            return
        past, _ = self._group_steps(cache, chunk, bits, frame, fg['steps'])
        for j in range(k):
            fg['emb'][j].copy_(embs[j])
            torch.add(fg['arange'], past[j], out=fg['pos'][j][0])
        fg['graph'].replay()

    def _capture_group(self, cache, embs, bits, frame):
        chunk, k = embs[0].shape[1], len(embs)
        static_emb = [e.clone() for e in embs]
        arange = torch.arange(chunk, device=self.device)
        pos = [torch.empty((1, chunk), dtype=torch.long, device=self.device) for _ in range(k)]
        past, steps = self._group_steps(cache, chunk, bits, frame, [None] * k)
        for j in range(k):
            torch.add(arange, past[j], out=pos[j][0])
        layers = self.text.layers
        done = [[torch.cuda.Event() for _ in layers] for _ in range(k - 1)]  # frame j's layer l has finished
        streams = [torch.cuda.Stream(device=self.device) for _ in range(k - 1)]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        hooks = []
        try:
            with torch.cuda.graph(graph):
                first = torch.cuda.current_stream()
                for st in streams:
                    st.wait_stream(first)  # the fork: the other forwards join the capture here
                for j in range(k):
                    stream = first if j == 0 else streams[j - 1]
                    if j > 0:  # layer l after the previous frame's layer l
                        hooks += [m.register_forward_pre_hook(
                            lambda mod, inp, l=l, ev=done[j - 1], st=stream: st.wait_event(ev[l]))
                            for l, m in enumerate(layers)]
                    if j < k - 1:
                        hooks += [m.register_forward_hook(lambda mod, inp, out, l=l, ev=done[j]: ev[l].record())
                                  for l, m in enumerate(layers)]
                    cache.begin_graph_steps(chunk, steps=steps[j])
                    with torch.cuda.stream(stream):
                        self.text(inputs_embeds=static_emb[j], past_key_values=cache, use_cache=True,
                                  position_ids=pos[j], attention_mask=None, return_dict=True)
                    cache.end_graph_steps()
                    for h in hooks:
                        h.remove()
                    hooks = []
                for st in streams:
                    first.wait_stream(st)
        finally:
            for h in hooks:
                h.remove()
            cache.end_graph_steps()
        for st in steps:
            st.upload()  # the jobs now carry the K/V addresses recorded in the graph
        graph.replay()
        self._group_graphs[self._graph_key(cache, chunk, k)] = dict(graph=graph, steps=steps, emb=static_emb, pos=pos, arange=arange,
                                              events=done, streams=streams)

    def _fork_forward(self, branch, ids, logits, lengths=None):
        """fp32 logits of the last `logits` positions of one forward on a fork of the decoder's
        reused cache. `lengths` splits the chunk into continuations of the fork's history, each
        with its own positions and attending to itself only (a block-diagonal chunk mask). With
        graphs=True a shape seen before replays a captured forward + lm_head (captured the second
        time it is seen; the first run is eager and warms the library paths)."""
        emb = self.text.get_input_embeddings()(ids.to(self.device))
        chunk = emb.shape[1]
        lengths = list(lengths) if lengths else None
        segments, rel = None, None
        if lengths:
            segments = [0]
            for n in lengths:
                segments.append(segments[-1] + n)
            rel = torch.cat([torch.arange(n, device=self.device) for n in lengths])
        else:
            rel = torch.arange(chunk, device=self.device)
        key = (chunk, int(logits), tuple(lengths) if lengths else None)
        if branch.sparse_blocks:
            key += (branch.sparse_blocks,)
        graphed = self.graphs and self._cache is not None and branch.arena is self._cache.arena
        if not graphed or key not in self._qa_seen:
            if graphed:
                self._qa_seen.add(key)
            past = self._position(branch)
            branch.chunk_segments = segments
            try:
                return self.forward(branch, embeddings=emb, positions=rel + past, logits=logits)
            finally:
                branch.chunk_segments = None
        fg = self._captured(self._qa_graphs, key, branch)
        steps = fg['steps'] if fg else None
        branch.begin_graph_steps(chunk, q_heads=None if fg else self.config.num_attention_heads, steps=steps)
        try:
            past = self._position(branch, branch.graph_step())
            if fg is None:
                static_emb, pos = emb.clone(), torch.empty((1, chunk), dtype=torch.long, device=self.device)
                torch.add(rel, past, out=pos[0])
                branch.chunk_segments = segments
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    out = self.text(inputs_embeds=static_emb, past_key_values=branch, use_cache=True,
                                    position_ids=pos, attention_mask=None, return_dict=True)
                    lg = self.model.lm_head(out.last_hidden_state[:, -int(logits):]).float()
                fg = self._qa_graphs[key] = dict(graph=graph, steps=branch._graph, emb=static_emb, pos=pos,
                                                 rel=rel.clone(), logits=lg)
                fg['steps'].upload()  # the jobs now carry the K/V addresses recorded in the graph
            else:
                fg['emb'].copy_(emb)
                torch.add(fg['rel'], past, out=fg['pos'][0])
            fg['graph'].replay()
            return fg['logits'].clone()
        finally:
            branch.chunk_segments = None
            branch.end_graph_steps()

    @staticmethod
    def _mean_loglik(logits, targets):
        return logits.log_softmax(-1).gather(1, targets[:, None]).mean()

    @torch.inference_mode()
    def generate(self, cache, question_ids, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, blocks=0):
        """Continues the question on a fork: one token for each random number of u [n] (gpu_ops.sample: fp32
        or fp64, on the decoder's device), int64 [n]. With `blocks` the question and every token attend to the
        tiles of the history that score highest for them, that many each, and to all that came after the
        question (GPUCache.attend_sparse; the cache's index is brought up to date first). From a row without a
        token that can be drawn on the tokens are -1. Nothing waits for the GPU, so a caller that stops at a
        token looks for it afterwards."""
        if u.dim() != 1:
            raise ValueError('generate expects one random number a token, u [n]')
        if blocks:
            cache.index()
        branch, ids, tokens = cache.fork(), question_ids, []
        branch.sparse_blocks = blocks
        for i in range(u.shape[0]):
            logits = self._fork_forward(branch, ids, 1)[0]
            tokens.append(sample(logits, u[i:i + 1], temperature, top_k, top_p, min_p))
            ids = tokens[-1][None].clamp(min=0)  # (-1 is no index into the embeddings)
        if not tokens:
            return u.new_empty(0, dtype=torch.int64)
        out = torch.cat(tokens)
        return out.masked_fill((out < 0).cumsum(0) > 0, -1)

    def _current(self):
        """The decoder's device as the current one: where a capture records and the fused layers launch."""
        return torch.cuda.device(self.device) if self.device.type == 'cuda' else contextlib.nullcontext()

    def _paged_forward(self, step, ids, last):
        """fp32 logits [sequences, vocabulary] of a step's tokens ids [1, tokens] at the places `last` of them."""
        out = self.text(inputs_embeds=self.text.get_input_embeddings()(ids), past_key_values=step, use_cache=True,
                        position_ids=step.positions[None], attention_mask=None, return_dict=True)
        return self.model.lm_head(out.last_hidden_state[0, last]).float()

    @torch.inference_mode()
    def generate_batch(self, pages, seqs, questions, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        """Continues each question [1, n] (of any lengths) on a branch of its sequence of the PagedCache `pages` (one
        of seqs each, or one for all; questions about one sequence attend to it together where they stand next to
        each other): tokens int64 [questions, n] for the random numbers u [questions, n], each row as generate() draws
        it. The branches take pages for a question and its tokens, and end with the call. Threads may call at once with one
        `pages` on one stream. With graphs=True the forwards of more than GRAPH_TOKENS tokens are replays of a captured one from
        the third token's on, the call waits for the GPU, and a capture allows no other thread's work on the device."""
        questions = list(questions)
        seqs = list(seqs) if hasattr(seqs, '__len__') else [seqs] * len(questions)
        if len(seqs) != len(questions) or u.dim() != 2 or u.shape[0] != len(questions):
            raise ValueError(f'generate_batch expects a sequence and random numbers u [questions, n] for each question, got '
                             f'{len(seqs)} and {list(u.shape)} for {len(questions)}')
        if any(x.dim() != 2 or x.shape[0] != 1 or not x.shape[1] for x in questions):
            raise ValueError('generate_batch expects questions of one token or more, [1, n]')
        if not u.numel():
            return u.new_empty(u.shape, dtype=torch.int64)
        branches, tokens, graph = [], [], None
        try:
            i = 0
            while i < len(seqs):  # branches of one sequence with one call
                n = next((j for j in range(i, len(seqs)) if seqs[j] != seqs[i]), len(seqs)) - i
                branches += pages.fork(seqs[i], n)
                i += n
            counts = [x.shape[1] for x in questions]
            last = torch.tensor(counts).cumsum(0).sub(1).to(self.device)
            ids = torch.cat([x.to(self.device) for x in questions], dim=1)
            # (a plan and the launches over it: another thread's call frees or moves no pages between the two)
            with pages.lock, self._current():
                step = pages.step(branches, counts)
                logits = self._paged_forward(step, ids, last)
            n, last = u.shape[1], slice(None)
            for i in range(n):
                tokens.append(sample(logits, u[:, i], temperature, top_k, top_p, min_p))
                if i + 1 == n:
                    break
                ids = tokens[-1][None].clamp(min=0)  # (-1 is no index into the embeddings)
                with pages.lock, self._current():
                    step = step.advance() if i else pages.step(branches, reserve=n)
                    if graph is not None:
                        held.copy_(ids)
                        graph.replay()
                    elif not (self.graphs and i and n > GRAPH_TOKENS):  # (the first of these forwards warms the library paths that a capture records)
                        logits = self._paged_forward(step, ids, last)
                    else:
                        held, graph = ids.clone(), torch.cuda.CUDAGraph()
                        torch.cuda.synchronize()
                        with torch.cuda.graph(graph):
                            logits = self._paged_forward(step, held, last)
                        graph.replay()
        finally:
            if graph is not None:
                torch.cuda.synchronize(self.device)  # (it may still run, and ends here)
            if branches:
                pages.free(branches)
        out = torch.stack(tokens, dim=1)
        return out.masked_fill((out < 0).cumsum(1) > 0, -1)

    @torch.inference_mode()
    def answer(self, cache, question_ids, candidates):
        """Mean token log-likelihood of each candidate on its own fork (src/streaming.py:209-225)."""
        scores = []
        for cand in candidates:
            ids = torch.cat((question_ids, cand), dim=1).to(self.device)
            branch = cache.fork()
            lg = self._fork_forward(branch, ids, cand.shape[1] + 1)
            scores.append(self._mean_loglik(lg[0, :-1], cand[0].to(self.device)))
        return torch.stack(scores)

    @torch.inference_mode()
    def answer_labels(self, cache, question_ids, label_ids):
        """The reference's 'label' protocol (src/streaming.py:202-208): one forward of the question
        on a fork; the scores are the last position's logits at the option-label token ids."""
        branch = cache.fork()
        logits = self._fork_forward(branch, question_ids, 1)[0, -1]
        return logits[torch.as_tensor(label_ids, device=self.device)]

    @torch.inference_mode()
    def prior_scores(self, prefix_ids, question_ids, candidates):
        """Candidate scores without the video, for the 'candidate_calibrated' protocol
        (src/streaming.py:124-127, 226-233): the same scoring on a cache holding only the prefix.
        Calibrated scores are answer(...) - prior_scores(...)."""
        total = prefix_ids.shape[1] + question_ids.shape[1] + max(c.shape[1] for c in candidates) + 64
        cache = self.create_cache(total)
        cache.select(16, -1)
        self.forward(cache, ids=prefix_ids)
        return self.answer(cache, question_ids, candidates)

    @torch.inference_mode()
    def answer_batched(self, cache, question_ids, candidates):
        """The same scores with the question once and all candidates in one block-diagonal chunk."""
        branch = cache.fork()
        q_logits = self._fork_forward(branch, question_ids, 1)[0]  # predicts each candidate's first token
        ids = torch.cat(candidates, dim=1)
        bounds = [0]
        for cand in candidates:
            bounds.append(bounds[-1] + cand.shape[1])
        # every candidate continues the question: positions restart at the fork's length for each
        lg = self._fork_forward(branch, ids, ids.shape[1], lengths=[c.shape[1] for c in candidates])[0]
        scores = []
        for i, cand in enumerate(candidates):
            pred = torch.cat((q_logits, lg[bounds[i]:bounds[i + 1] - 1]), 0)
            scores.append(self._mean_loglik(pred, cand[0].to(self.device)))
        return torch.stack(scores)
