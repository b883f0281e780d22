from __future__ import annotations

from abc import ABC, abstractmethod

import torch

from ..layers import BaseOP


class BaseLLMModel(ABC, BaseOP):
    _weights_loaded = 0  # how often weights were loaded

    @abstractmethod
    def forward(self) -> torch.Tensor: ...

    def on_weights_loaded(self) -> None:
        self._weights_loaded += 1

    @property
    def graph_key(self) -> tuple:
        """What a forward depends on besides its batch. Whoever keeps captured graphs of it, or
        K/V that it wrote, drops them when this changes."""
        return (self._weights_loaded,)
