"""Encoders: thermometer (real features), embedding (token ids) and their base class."""

from .base_encoder import BaseEncoder
from .embedding import EmbeddingEncoder, embedding_lookup
from .thermometer import DistributiveThermometerEncoder, GaussianThermometerEncoder, ThermometerEncoder

__all__ = ["BaseEncoder", "ThermometerEncoder", "GaussianThermometerEncoder", "DistributiveThermometerEncoder",
           "EmbeddingEncoder", "embedding_lookup"]
