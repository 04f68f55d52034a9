"""Latent KV cache for MLA decode: drop-in for src/kernels/mla_cache.py:29-219.

Same constructor, properties (`current_len`, `remaining_capacity`, `memory_bytes`), methods
(`update`, `get`, `reset`, `for_inference`) and error messages as the reference's
LatentKVCache: per sequence and position it stores the raw, pre-norm 512-wide latent
(`kv_latent`) and the raw, un-rotated 64-wide k_pe (`k_pe_cache`), pre-allocated to
`max_seq`, written at the current length and read back as zero-copy views.

On a CUDA device it also keeps two side arrays for the decode kernel
(ds_kernels.mla_decode_step): `rstd` (f32 [bsz, max_seq]: the latent RMSNorm's row scale
rsqrt(mean(latent^2) + eps)) and `k_pe_rot` (bf16 [bsz, max_seq, 64]: k_pe rotated at its
position).  The fused paths (FusedMLA.prefill / FusedMLA.decode) write them together with the
raw values; positions written through the reference's `update()` (which has no RoPE tables)
get them on the next decode step.  `memory_bytes` counts the two reference buffers, as the
reference does; `side_bytes` the side arrays.
"""
from __future__ import annotations

import weakref
from typing import Optional, Tuple

import torch

_capturing = torch.cuda.is_current_stream_capturing


class LatentKVCache:
    def __init__(self, bsz: int, max_seq: int, kv_lora_rank: int = 512, rope_head_dim: int = 64,
                 device: str = "cuda", dtype: torch.dtype = torch.bfloat16):
        if not isinstance(bsz, int) or bsz < 1:
            raise ValueError(f"bsz must be a positive integer, got {bsz}")
        if not isinstance(max_seq, int) or max_seq < 1:
            raise ValueError(f"max_seq must be a positive integer, got {max_seq}")
        self.bsz = bsz
        self.max_seq = max_seq
        self.kv_lora_rank = kv_lora_rank
        self.rope_head_dim = rope_head_dim
        self.device = torch.device(device)
        self.dtype = dtype
        self._len = 0
        self.kv_latent = torch.zeros((bsz, max_seq, kv_lora_rank), dtype=dtype, device=self.device)
        self.k_pe_cache = torch.zeros((bsz, max_seq, rope_head_dim), dtype=dtype, device=self.device)
        # side arrays of the decode kernel (CUDA only); valid for positions < _side_len
        self._side_len = 0
        if self.device.type == "cuda":
            self.rstd = torch.zeros((bsz, max_seq), dtype=torch.float32, device=self.device)
            self.k_pe_rot = torch.zeros((bsz, max_seq, rope_head_dim), dtype=dtype,
                                        device=self.device)
            # the length on the device: the decode kernels read the position from it and
            # advance it, so a captured CUDA graph of a decode step replays at successive
            # positions (the host-side length is advanced alongside)
            self.len_dev = torch.zeros((1,), dtype=torch.int32, device=self.device)
        else:
            self.rstd = self.k_pe_rot = self.len_dev = None

    # ---- properties (reference surface) --------------------------------------------------
    @property
    def current_len(self) -> int:
        """Number of tokens currently stored in the cache."""
        return self._len

    @property
    def remaining_capacity(self) -> int:
        """Number of additional tokens that can be appended."""
        return self.max_seq - self._len

    @property
    def memory_bytes(self) -> int:
        """Total bytes consumed by both cache buffers."""
        return (self.kv_latent.numel() + self.k_pe_cache.numel()) * self.kv_latent.element_size()

    @property
    def side_bytes(self) -> int:
        """Bytes of the decode kernel's side arrays (0 off CUDA)."""
        if self.rstd is None:
            return 0
        return self.rstd.numel() * 4 + self.k_pe_rot.numel() * self.k_pe_rot.element_size()

    # ---- core operations (reference surface) ---------------------------------------------
    def update(self, compressed_kv: torch.Tensor, k_pe: torch.Tensor) -> None:
        """Append new tokens: compressed_kv [bsz, new_tokens, kv_lora_rank], k_pe
        [bsz, new_tokens, rope_head_dim] (the raw k_pe, without the head dim)."""
        if compressed_kv.dim() != 3:
            raise ValueError(
                f"compressed_kv must be 3D [bsz, new_tokens, kv_lora_rank], "
                f"got shape {tuple(compressed_kv.shape)}")
        if k_pe.dim() != 3:
            raise ValueError(
                f"k_pe must be 3D [bsz, new_tokens, rope_head_dim], got shape {tuple(k_pe.shape)}")
        new_tokens = compressed_kv.shape[1]
        if self._len + new_tokens > self.max_seq:
            raise RuntimeError(
                f"KV cache overflow: current_len={self._len}, new_tokens={new_tokens}, "
                f"max_seq={self.max_seq}. Increase max_seq or reset the cache.")
        slot = slice(self._len, self._len + new_tokens)
        self.kv_latent[:, slot, :] = compressed_kv.to(self.device, self.dtype)
        self.k_pe_cache[:, slot, :] = k_pe.to(self.device, self.dtype)
        self._len += new_tokens
        if self.len_dev is not None:
            self.len_dev.fill_(self._len)

    def get(self, seq_len: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """(kv_latent [bsz, seq_len, kv_lora_rank], k_pe [bsz, seq_len, rope_head_dim]) views."""
        if seq_len is None:
            seq_len = self._len
        if seq_len > self._len:
            raise ValueError(f"Requested seq_len={seq_len} but cache only has {self._len} tokens.")
        return self.kv_latent[:, :seq_len, :], self.k_pe_cache[:, :seq_len, :]

    def reset(self) -> None:
        """Clear the cache for a new sequence (keeps the memory)."""
        self._len = 0
        self._side_len = 0
        if self.len_dev is not None:
            self.len_dev.zero_()

    def __repr__(self) -> str:
        used_mb = (self._len * (self.kv_lora_rank + self.rope_head_dim)
                   * self.kv_latent.element_size() * self.bsz) / (1024 ** 2)
        total_mb = self.memory_bytes / (1024 ** 2)
        return (f"LatentKVCache(bsz={self.bsz}, tokens={self._len}/{self.max_seq}, "
                f"used={used_mb:.2f}MB/{total_mb:.2f}MB, device={self.device}, dtype={self.dtype})")

    @classmethod
    def for_inference(cls, bsz: int, max_seq: int = 4096, device: str = "cuda") -> "LatentKVCache":
        """BF16 cache with the production defaults (512-wide latent, 64-wide k_pe)."""
        return cls(bsz=bsz, max_seq=max_seq, kv_lora_rank=512, rope_head_dim=64, device=device,
                   dtype=torch.bfloat16)

    # ---- decode-kernel bookkeeping ----------------------------------------------------------
    def _require_decode_layout(self) -> None:
        if self.rstd is None or self.dtype != torch.bfloat16 or self.kv_lora_rank != 512 \
                or self.rope_head_dim != 64:
            raise RuntimeError("the fused MLA kernels need a bf16 CUDA cache with a 512-wide "
                               "latent and a 64-wide k_pe")

    def _sync_side(self, cos: torch.Tensor, sin: torch.Tensor, eps: float) -> None:
        """Fill the side arrays of positions written through update() (raw values only)."""
        self._require_decode_layout()
        if self._side_len < self._len:
            import ds_kernels
            s0, s1 = self._side_len, self._len
            ds_kernels.mla_cache_append(self.kv_latent[:, s0:s1], self.k_pe_cache[:, s0:s1], self,
                                        s0, cos, sin, eps, copy_raw=False)
            self._side_len = s1

    def _advance(self, n: int, device_counted: bool) -> None:
        """A fused kernel appended n tokens, side arrays included (the callers bring the side
        arrays of earlier positions up to date before they launch); device_counted: the
        kernels already advanced len_dev."""
        if self._side_len < self._len:
            raise RuntimeError("LatentKVCache: side arrays were stale when tokens were appended")
        self._len += n
        self._side_len = self._len
        if not device_counted:
            self.len_dev.fill_(self._len)


class LatentKVCache4:
    """Latent KV cache held in 4 bits: 310 bytes a token against LatentKVCache's 1156 (with its
    side arrays).  Filled by ds_kernels.mla_cache4_append (FusedMLA.prefill / decode), read by
    ds_kernels.mla_decode_attention4, trimmed by ds_kernels.mla_cache4_evict.

    Sequences have their own lengths (device, int32 `lens`) and next positions (`next_pos`: the
    tokens seen, evicted ones included, so a token keeps its rotary position when others leave).
    Arrays, per sequence and slot (`slots` = max_seq rounded up to 64):

        codes   uint8 [bsz, slots, 288]  two 4-bit codes a byte, low half first: 512 dimensions
                                         of the raw latent, then 64 of k_pe rotated at its
                                         position; value = (code - 8) * scale of its group
        scales  bf16  [bsz, 5, slots]    four groups of 128 latent dimensions, then k_pe:
                                         bf16(max |v| / 7)
        rstd    f32   [bsz, slots]       rsqrt(mean(latent^2) + eps) of the exact latent
        pos     int32 [bsz, slots]       position of the token in the slot
        mass    f32   [bsz, slots]       accumulated attention weight: 0 for a token that is
                                         appended (prompts too), moved by decode steps alone

    The host knows only a bound on the lengths (`current_len`: exact for batches that are not
    ragged), which it advances with every call; no call synchronises.  A call recorded into a
    CUDA graph takes the whole cache as its bound, so replays may go on to the last slot; replays
    move the device-side lengths only, and the caller reports them with note_replay().  A replayed
    token that finds no slot is dropped, and one whose position lies behind the RoPE tables is
    rotated as their last row: who replays compares current_len with max_seq, and positions with
    the tables, as FusedDecoderStack.replay_decode does."""

    def __init__(self, bsz: int, max_seq: int, device="cuda"):
        if not isinstance(bsz, int) or bsz < 1:
            raise ValueError(f"bsz must be a positive integer, got {bsz}")
        if not isinstance(max_seq, int) or max_seq < 1:
            raise ValueError(f"max_seq must be a positive integer, got {max_seq}")
        self.bsz, self.max_seq = bsz, max_seq
        self.slots = -(-max_seq // 64) * 64
        dev = torch.device(device)
        self._codes = torch.zeros((bsz, self.slots, 288), dtype=torch.uint8, device=dev)
        dev = self._codes.device
        self._scales = torch.zeros((bsz, 5, self.slots), dtype=torch.bfloat16, device=dev)
        self._rstd = torch.zeros((bsz, self.slots), dtype=torch.float32, device=dev)
        self._pos = torch.zeros((bsz, self.slots), dtype=torch.int32, device=dev)
        self._mass = torch.zeros((bsz, self.slots), dtype=torch.float32, device=dev)
        # lengths, next positions, and a row of counters that are zero between calls
        self._state = torch.zeros((3, bsz), dtype=torch.int32, device=dev)
        self._bind()
        self._bound = 0      # no sequence is longer
        self._seen = 0       # no next position is larger
        # (the two are those behind a recorded reset or eviction; until it is replayed the cache
        # holds what it held, and this pair bounds that)
        self._held: Optional[Tuple[int, int]] = None

    # the arrays may be written into, but not replaced: launches take their addresses
    codes = property(lambda self: self._codes)
    scales = property(lambda self: self._scales)
    rstd = property(lambda self: self._rstd)
    pos = property(lambda self: self._pos)
    mass = property(lambda self: self._mass)
    state = property(lambda self: self._state)
    lens = property(lambda self: self._lens)
    next_pos = property(lambda self: self._next_pos)

    def _bind(self) -> None:
        self.device = self._codes.device
        self.index = self._codes.get_device()    # the CUDA device's ordinal, -1 off CUDA
        self._lens, self._next_pos = self._state[0], self._state[1]
        # the addresses as the C entry points take them
        self._ptrs = tuple(t.data_ptr() for t in (self._codes, self._scales, self._rstd, self._pos,
                                                  self._mass, self._state))

    _source = None  # the cache that a recorded eviction into this one reads, as a weak reference

    def __getstate__(self) -> dict:  # no graph evicts into a copy
        return {**self.__dict__, "_source": None}

    def __setstate__(self, state: dict) -> None:  # a deep copy's or a pickle's arrays are others
        self.__dict__.update(state)
        self._bind()

    @property
    def current_len(self) -> int:
        """A bound on the sequences' lengths (the length itself when they are equal)."""
        return self._now()[0]

    @property
    def remaining_capacity(self) -> int:
        """Tokens that surely still fit into every sequence."""
        return self.max_seq - self.current_len

    @property
    def memory_bytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in
                   (self.codes, self.scales, self.rstd, self.pos, self.mass, self.state))

    @property
    def bound_for_launch(self) -> int:
        """The bound that a launch is sized for: all slots inside a graph capture, because a
        replay sees later lengths."""
        return self.max_seq if _capturing() else self.current_len

    def reset(self) -> None:
        """Clear the cache for new sequences (keeps the memory)."""
        import ds_kernels
        ds_kernels.mla_cache4_reset(self)
        self._hold()
        self._bound = self._seen = 0

    def get(self, seq_len: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """(raw latent bf16 [bsz, seq_len, 512], rotated k_pe bf16 [bsz, seq_len, 64]) as the
        codes stand for them; zeros from a sequence's length on."""
        import ds_kernels
        lat, kpe = ds_kernels.mla_cache4_get(self, seq_len)
        return lat, kpe

    def evict(self, budget: int, recent: int = 0, out: "Optional[LatentKVCache4]" = None):
        """ds_kernels.mla_cache4_evict on this cache."""
        import ds_kernels
        return ds_kernels.mla_cache4_evict(self, budget, recent, out)

    def note_replay(self, tokens: int = 1, budget: Optional[int] = None,
                    src: "Optional[LatentKVCache4]" = None) -> None:
        """A replayed graph appended `tokens` tokens to every sequence, and before (or after) it
        evicted them down to `budget` slots (0: cleared them).  If the eviction read another cache,
        the bound is the whole budget, whatever that one holds; with the other cache named as `src`
        it is what `src` is bounded by now.  Notes on several caches go in the order of the
        graph's work."""
        if budget is not None:
            bound, seen = self._now()
            if budget <= 0:
                bound = seen = 0
            elif src is not None:
                bound, seen = src._now()
            elif self._source is not None:
                other = self._source()
                bound, seen = budget, max(seen, other._now()[1] if other is not None else 0)
            self._bound, self._seen, self._held = min(bound, budget), seen, None
        self._advance(tokens)

    # ---- saving and restoring ------------------------------------------------------------
    def state_dict(self) -> dict:
        """Copies of everything the cache holds."""
        return {k: getattr(self, k).clone()
                for k in ("codes", "scales", "rstd", "pos", "mass", "lens", "next_pos")}

    def load_state_dict(self, state: dict) -> None:
        """Take over saved contents (same batch; the saved slots may be fewer).  `codes`,
        `scales`, `rstd` and `lens` are needed; without `pos` slot i holds position i, without
        `next_pos` it is the length, without `mass` the weights are 0.  Synchronises once to
        read the largest length."""
        for k in ("codes", "scales", "rstd", "lens"):
            if k not in state:
                raise ValueError(f"load_state_dict: {k} is missing")
        n = state["codes"].shape[1]
        want = {"codes": (self.bsz, n, 288), "scales": (self.bsz, 5, n), "rstd": (self.bsz, n),
                "pos": (self.bsz, n), "mass": (self.bsz, n), "lens": (self.bsz,),
                "next_pos": (self.bsz,)}
        for k, t in state.items():
            if k not in want or tuple(t.shape) != want[k]:
                raise ValueError(f"load_state_dict: unexpected {k} of shape {tuple(t.shape)}")
        lens = state["lens"].to(self.device, torch.int32)
        nxt = state["next_pos"].to(self.device, torch.int32) if "next_pos" in state else lens
        early = (nxt < lens).any().to(torch.int32)
        lo, hi, top, early = (int(v) for v in
                              torch.stack([lens.min(), lens.max(), nxt.max(), early]).tolist())
        if n > self.slots or lo < 0 or hi > min(n, self.max_seq):
            raise ValueError("load_state_dict: the saved sequences do not fit the cache")
        if early:
            raise ValueError("load_state_dict: next_pos must be at least the number of tokens")
        for k in ("codes", "scales", "rstd"):
            dst = getattr(self, k)
            (dst[:, :, :n] if k == "scales" else dst[:, :n]).copy_(state[k])
        if "pos" in state:
            self.pos[:, :n].copy_(state["pos"])
        else:
            self.pos.copy_(torch.arange(self.slots, dtype=torch.int32, device=self.device)
                           .expand(self.bsz, -1))
        if "mass" in state:
            self.mass[:, :n].copy_(state["mass"])
        else:
            self.mass.zero_()
        self.lens.copy_(lens)
        self.next_pos.copy_(nxt)
        self._bound, self._seen, self._held = hi, top, None

    def __repr__(self) -> str:
        return (f"LatentKVCache4(bsz={self.bsz}, tokens<={self.current_len}/{self.max_seq}, "
                f"memory={self.memory_bytes / 2 ** 20:.2f}MB, device={self.device})")

    # ---- bookkeeping of the fused calls --------------------------------------------------
    def _recording(self) -> bool:
        return self.index >= 0 and _capturing()

    def _now(self) -> Tuple[int, int]:
        """Bounds on the lengths and next positions that the next call meets."""
        if self._held is not None and not self._recording():
            return self._held
        return self._bound, self._seen

    def _hold(self) -> None:
        """Before the contents are replaced: recorded into a graph, they stay until a replay, and
        the calls up to then count on what is there."""
        if not self._recording():
            self._held = None
        elif self._held is None:
            self._held = self._bound, self._seen

    def _check_room(self, n: int, table_rows: int) -> None:
        bound, seen = self._now()
        if bound + n > self.max_seq:
            raise RuntimeError(
                f"KV cache overflow: current_len={bound}, new_tokens={n}, "
                f"max_seq={self.max_seq}. Increase max_seq, evict or reset the cache.")
        if seen + n > table_rows:
            raise RuntimeError(f"LatentKVCache4: position {seen + n - 1} is beyond the RoPE "
                               f"tables ({table_rows} positions)")

    def _advance(self, n: int) -> None:
        if self._held is not None and n > 0 and not self._recording():
            self._held = min(self._held[0] + n, self.max_seq), self._held[1] + n
            return
        # (n < 0: what a recording has counted too many)
        self._bound = min(self._bound + n, self.max_seq)
        self._seen += n

    def _evicted(self, src: "LatentKVCache4", budget: int) -> None:
        bound, seen = src._now()
        bound = min(bound, budget)
        self._hold()
        if src is not self and self._recording():  # a replay takes what src holds by then
            self._source = weakref.ref(src)
            bound = budget
        self._bound, self._seen = bound, seen
