# Builds the gfx950 C-ABI library in-tree (the .so travels to the GPU box with the snapshot).
HIPCC ?= /opt/rocm/bin/hipcc
ARCH ?= gfx950
PKG := d-vae_amd
CSRC := $(PKG)/csrc
LIB := $(PKG)/lib/libdvae_hip.so
LEARN_HDRS := $(CSRC)/layer_norm.hpp $(CSRC)/newton_schulz.hpp $(CSRC)/newton_schulz_small.hpp
HDRS := $(filter-out $(LEARN_HDRS),$(wildcard $(CSRC)/*.hpp)) include/dvae_hip.h
# No packed fp32 arithmetic in the kernels: some of its forms have given wrong results now and then (the host pass does not know
# the feature and says so).
FLAGS := --offload-arch=$(ARCH) -O3 -std=c++17 -fPIC -fno-gpu-rdc -Wall -Wno-unused-function -mllvm -pragma-unroll-threshold=1000000 \
    -Xclang -target-feature -Xclang -packed-fp32-ops

all: $(LIB)

$(PKG)/lib/dvae_hip.o: $(CSRC)/dvae_hip.hip $(HDRS)
	@mkdir -p $(PKG)/lib
	$(HIPCC) $(FLAGS) -c -o $@ $<

$(PKG)/lib/dvae_learn.o: $(CSRC)/dvae_learn.hip $(CSRC)/common.hpp $(LEARN_HDRS) include/dvae_hip.h
	@mkdir -p $(PKG)/lib
	$(HIPCC) $(FLAGS) -c -o $@ $<

$(LIB): $(PKG)/lib/dvae_hip.o $(PKG)/lib/dvae_learn.o
	$(HIPCC) --offload-arch=$(ARCH) -fPIC -shared -fno-gpu-rdc -o $@ $^

clean:
	rm -f $(LIB) $(PKG)/lib/dvae_hip.o $(PKG)/lib/dvae_learn.o

.PHONY: all clean
