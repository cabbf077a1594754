// plumbing.cpp — the two "plumbing" configurations of SURVEY.md §8a next to the NeRF path: P1 image fitting (src/testbed_image.cu) and P2 SDF fitting
// (the training step of src/testbed_sdf.cu:1229-1252 on user-provided samples).  Both are a tcnn NetworkWithInputEncoding — HashGrid over 2 / 3
// dimensions -> FullyFusedMLP 64 x 2 hidden -> 16 — trained by Trainer::training_step + optimizer_step(128); here: ngp_hip_gridmlp_* + ngp_hip_loss_and_gradient
// + the same Adam / ExponentialDecay / Ema kernel as the NeRF path, on the Testbed's own parameter / optimizer buffers.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>

#include "image_io.h"
#include "snapshot.h"
#include "testbed.h"

namespace ngp {

#define HIP_TRY(x) do { hipError_t e_ = (x); if (e_ != hipSuccess) throw std::runtime_error(std::string(#x) + ": " + hipGetErrorString(e_)); } while (0)
static constexpr float LOSS_SCALE = 128.0f;                 // testbed.h:272, optimizer_step(stream, 128)
static constexpr uint32_t BATCH_SIZE_GRANULARITY = 128;     // tcnn::batch_size_granularity
static inline uint32_t next_multiple(uint32_t v, uint32_t m) { return (v + m - 1) / m * m; }

void Testbed::reset_network_gridmlp() {  // testbed.cu:2249-2470, Image / Sdf branch (2397-2445)
	join_side_ema();
	const Json& config = m_network_config;
	const Json empty = Json::object();
	const Json& enc = config.contains("encoding") ? config["encoding"] : empty;
	// what may be refused is read first: a refusal leaves the network, and what says how its parameters lie, as they were
	auto require = [](bool ok, const std::string& what) { if (!ok) throw std::runtime_error{"network config not supported by the gfx950 fused kernels: " + what}; };
	std::string enc_type = enc.value("otype", "HashGrid"); std::transform(enc_type.begin(), enc_type.end(), enc_type.begin(), ::tolower);
	require(enc_type == "hashgrid", "encoding.otype must be HashGrid");
	require((uint32_t)enc.value("n_features_per_level", 2) == 2 && (uint32_t)enc.value("n_levels", 16) == 16, "HashGrid must have 16 levels x 2 features");
	std::string net_type = config.contains("network") ? config["network"].value("otype", "FullyFusedMLP") : std::string("FullyFusedMLP"); std::transform(net_type.begin(), net_type.end(), net_type.begin(), ::tolower);
	const bool gated = net_type == "gatedmlp";
	NgpGatedFfn block{};
	if (gated) {
		const Json& net = config["network"];
		const int width = (int)net.value("n_neurons", 64);
		require(width >= 8 && width <= 65536 && width % 8 == 0, "GatedMLP: n_neurons must be a multiple of 8 up to 65536");
		require(net.value("n_hidden_layers", 1) == 1, "GatedMLP: n_hidden_layers must be 1");
		std::string act = net.value("activation", "SiLU"); std::transform(act.begin(), act.end(), act.begin(), ::tolower);
		block.activation = act == "silu" ? NGP_ACT_SILU : act == "gelu" ? NGP_ACT_GELU : act == "relu" ? NGP_ACT_RELU : act == "sigmoid" || act == "logistic" ? NGP_ACT_LOGISTIC : act == "none" ? NGP_ACT_NONE : -1;
		require(block.activation >= 0, "GatedMLP: activation must be SiLU, GELU, ReLU, Sigmoid or None");
		std::string out_act = net.value("output_activation", "None"); std::transform(out_act.begin(), out_act.end(), out_act.begin(), ::tolower);
		require(out_act == "none", "GatedMLP: output_activation must be None");
		block.n_in = 32; block.n_hidden = (uint32_t)width; block.n_out = 16; block.dtype = NGP_DTYPE_F16;
	} else if (config.contains("network")) require(config["network"].value("n_neurons", 64) == 64 && config["network"].value("n_hidden_layers", 2) == 2, "network must be 64 neurons x 2 hidden layers");
	std::string loss = config.contains("loss") ? config["loss"].value("otype", "L2") : std::string("L2");
	std::transform(loss.begin(), loss.end(), loss.begin(), ::tolower);
	ELossType loss_type;
	if (loss == "l2") loss_type = ELossType::L2;
	else if (loss == "relativel2") loss_type = ELossType::RelativeL2;
	else if (loss == "l1") loss_type = ELossType::L1;
	else if (loss == "mape") loss_type = ELossType::Mape;
	else throw std::runtime_error{"loss '" + loss + "' is not implemented for the grid -> MLP configs (L2, RelativeL2, L1, MAPE are)"};
	const uint32_t n_dims = gridmlp_n_dims();
	const uint32_t log2_hashmap_size = (uint32_t)enc.value("log2_hashmap_size", 15);
	uint32_t base_resolution = (uint32_t)enc.value("base_resolution", 0);
	if (!base_resolution) base_resolution = 1u << (log2_hashmap_size / n_dims);
	float desired_resolution = 2048.0f;   // finest level over the unit cube (2315); Image: half the image resolution (2317)
	if (m_testbed_mode == ETestbedMode::Image) desired_resolution = (float)std::max(m_image.resolution[0], m_image.resolution[1]) / 2.0f;
	float per_level_scale = (float)enc.value("per_level_scale", 0.0);
	if (per_level_scale <= 0.0f) per_level_scale = std::exp(std::log(desired_resolution * 1.0f / (float)base_resolution) / 15.0f);
	NgpNetDesc desc{};
	check(ngp_hip_gridmlp_make_desc_host(n_dims, 16, log2_hashmap_size, base_resolution, per_level_scale, &desc), "ngp_hip_gridmlp_make_desc_host");
	if (config.contains("optimizer")) parse_optimizer_config(config["optimizer"]);

	tuner_reset();
	m_rng = Pcg32(m_seed);
	m_windowless_render_surface.reset_accumulation();
	m_nerf.training.loss_type = loss_type;
	m_gated = gated;
	m_gated_block = block;
	m_num_levels = 16;
	m_base_grid_resolution = base_resolution;
	m_per_level_scale = per_level_scale;
	m_desc = desc;
	m_n_params = ngp_hip_gridmlp_n_params_host(&m_desc);
	m_n_matrix_params = NGP_GRIDMLP_N_PARAMS;
	m_matrices.clear();
	if (m_gated) {   // gate, up, down, grid
		const uint32_t f = m_gated_block.n_hidden;
		add_matrix(f, 32); add_matrix(f, 32); add_matrix(16, f);
		m_n_matrix_params = 80u * f;
		m_n_params = (size_t)m_n_matrix_params + 2u * (size_t)m_desc.n_grid_entries;
	} else { add_matrix(64, 32); add_matrix(64, 64); add_matrix(16, 64); }
	m_desc_gpu.resize(sizeof(NgpNetDesc));
	m_desc_gpu.copy_from_host(&m_desc, sizeof(NgpNetDesc));
	m_optimizer_step = 0;
	m_params.resize(m_n_params * 2); m_inference_params.resize(m_n_params * 2); m_grads.resize(m_n_params * 2);
	m_master.resize(m_n_params * 4); m_first_moments.resize(m_n_params * 4); m_second_moments.resize(m_n_params * 4); m_ema.resize(m_n_params * 4);
	m_first_moments.memset(0, m_stream); m_second_moments.memset(0, m_stream); m_ema.memset(0, m_stream); m_grads.memset(0, m_stream);
	if (m_gated) gated_init_params();
	else check(ngp_hip_gridmlp_init_params(m_stream, &m_desc, m_seed, m_master.as<float>(), m_params.as<uint16_t>(), m_inference_params.as<uint16_t>()), "ngp_hip_gridmlp_init_params");
	if (m_gated && m_dloss.bytes()) m_dloss.memset(0, m_stream);
	m_loss_scalar_gpu.resize(4);
	m_training_step = 0;
	m_loss_scalar = 0.f;
	sync();
}

// as the fused MLP's parameters start: uniform within sqrt(6 / (rows + columns)) per matrix (a down projection's 16 padded outputs counted), the grid within 1e-4, one number of the
// stream per parameter
void Testbed::gated_init_params() {
	std::vector<float> w(m_n_params);
	std::vector<uint16_t> h(m_n_params);
	Pcg32 rng(m_seed);
	size_t i = 0;
	auto fill = [&](size_t end, float scale) { for (; i < end; ++i) { w[i] = rng.next_float() * (2.0f * scale) - scale; h[i] = float_to_half_bits(w[i]); } };
	for (const NgpMuonMatrix& m : m_matrices) fill((size_t)m.offset + (size_t)m.rows * m.cols, std::sqrt(6.0f / (float)(m.rows + m.cols)));
	fill(m_n_params, 1e-4f);
	m_master.copy_from_host(w.data(), w.size() * 4);
	m_params.copy_from_host(h.data(), h.size() * 2);
	m_inference_params.copy_from_host(h.data(), h.size() * 2);
}

// rows of a gated block to a call where nothing has to be kept: 2^20 at most, and a hidden row's share of 1 GiB each (8192 rows of 65536 neurons)
uint32_t Testbed::gated_chunk() const { return std::min<uint32_t>(1u << 20, (1u << 29) / m_gated_block.n_hidden & ~255u); }

// encoding and block on n positions; x: their encoded features
void Testbed::gated_forward(const uint16_t* params, const float* pos, uint32_t n_dims, uint32_t n, uint16_t* out, uint16_t* x, DeviceBuffer& enc_ws, DeviceBuffer& gated_ws, const char* who) {
	enc_ws.enlarge(ngp_hip_nerf_encode_workspace_bytes(n));
	gated_ws.enlarge(std::max<uint64_t>(16, ngp_hip_gated_ffn_workspace_bytes(&m_gated_block, n, 0)));
	const uint32_t f = m_gated_block.n_hidden;
	check(ngp_hip_grid_encode(m_stream, n_dims, m_desc_gpu.as<NgpNetDesc>(), params + m_n_matrix_params, pos, n_dims, n, x, enc_ws.data(), enc_ws.bytes()), who);
	check(ngp_hip_gated_ffn_forward(m_stream, &m_gated_block, n, x, 32, params, params + 32 * f, params + 64 * f, out, gm_out_stride(), gated_ws.data(), gated_ws.bytes()), who);
}

// the network's outputs (rows of gm_out_stride()), nothing kept for a backward pass: rendering, errors, queries
void Testbed::gridmlp_inference(const uint16_t* params, const float* pos, uint32_t n_dims, uint32_t n, uint16_t* out, const char* who) {
	if (!m_gated) {
		check(ngp_hip_gridmlp_forward(m_stream, n_dims, m_desc_gpu.as<NgpNetDesc>(), params, pos, n_dims, n, out, gm_out_stride(), nullptr), who);
		return;
	}
	const uint32_t chunk = std::min(n, gated_chunk());
	m_gated_x.enlarge((size_t)chunk * 32 * 2);
	for (uint32_t first = 0; first < n; first += chunk)
		gated_forward(params, pos + (size_t)first * n_dims, n_dims, std::min(chunk, n - first), out + (size_t)first * gm_out_stride(), m_gated_x.as<uint16_t>(), m_gated_enc_ws, m_gated_infer_ws, who);
}

// What the loss is multiplied by, so that F16 holds the gradients: 128 as everywhere, per sample 1 / n of it.  A gated network needs more of it for a large batch: its features start
// within 1e-4 and a gate's gradient is a product with another of them, 1e-9 of a batch of 2^18 and so zero in F16 (the smallest is 6e-8): the image config stood at 3.03 dB for 1000
// steps, with 1024 or more it reaches 35 to 36.  From 2^14 samples on a sample's share stays what it is there, up to 2^20.  The weights' gradients, sums over the batch, grow with the
// scale: 8192 leaves them 8, so an L2 loss whose residuals are larger than one (its last value read; none before the first step, whose hidden values are 1e-9) gives that back, down
// to 128.  The relative losses keep 128: their gradients are up to 100 times as large, and at 2^20 samples 12 % (MAPE) and more of the table's first gradients are there.
float Testbed::gridmlp_loss_scale(uint32_t n) const {
	float scale = LOSS_SCALE;
	const bool l2 = m_nerf.training.loss_type == ELossType::L2;
	if (!m_gated || (!l2 && m_nerf.training.loss_type != ELossType::L1)) return scale;
	for (uint32_t k = n >> 15; k && scale < 64.0f * LOSS_SCALE; k >>= 1) scale *= 2.0f;
	for (float squares = l2 ? m_loss_scalar : 0.0f; squares > 1.0f && scale > LOSS_SCALE; squares *= 0.25f) scale *= 0.5f;
	return scale;
}

// Trainer::training_step (forward, loss, backward) + optimizer_step(128) + Trainer::loss (sum of the per-element values)
void Testbed::gridmlp_training_step(const float* pos, uint32_t n_dims, const float* targets, uint32_t dims, uint32_t n, bool get_loss_scalar) {
	if (n % 256) throw std::runtime_error{"training batch size must be a multiple of 256"};
	m_gm_out.enlarge((size_t)n * gm_out_stride() * 2); m_x_saved.enlarge((size_t)n * 32 * 2);
	const size_t dloss_bytes = (size_t)n * gm_out_stride() * 2;
	const bool grown = m_dloss.bytes() < dloss_bytes;
	m_dloss.enlarge(dloss_bytes);
	if (m_gated && grown) m_dloss.memset(0, m_stream);   // the loss writes channels 0..3 of the block's 16
	m_gm_values.enlarge((size_t)n * dims * 4);
	m_bwd_scratch.enlarge(ngp_hip_gridmlp_backward_scratch_bytes(n));
	const NgpNetDesc* desc = m_desc_gpu.as<NgpNetDesc>();
	profile_begin(PK_FORWARD);
	// fused or encode + MLP kernel: measured on this workload (testbed.h ENetworkPass) — random SDF points want the two-kernel pass, stratified image batches the fused one
	if (m_gated) gated_forward(m_params.as<uint16_t>(), pos, n_dims, n, m_gm_out.as<uint16_t>(), m_x_saved.as<uint16_t>(), m_enc_ws, m_gated_ws, "gated forward");
	else if (tuner_pick(m_stream)) {
		m_enc_ws.enlarge(ngp_hip_nerf_encode_workspace_bytes(n));
		check(ngp_hip_gridmlp_forward_ws(m_stream, n_dims, desc, m_params.as<uint16_t>(), pos, n_dims, n, m_gm_out.as<uint16_t>(), gm_out_stride(), m_x_saved.as<uint16_t>(), m_enc_ws.data(), m_enc_ws.bytes()), "gridmlp_forward (two kernels)");
	} else {
		check(ngp_hip_gridmlp_forward(m_stream, n_dims, desc, m_params.as<uint16_t>(), pos, n_dims, n, m_gm_out.as<uint16_t>(), gm_out_stride(), m_x_saved.as<uint16_t>()), "gridmlp_forward");
	}
	if (!m_gated) tuner_done(m_stream);
	profile_end(PK_FORWARD, n);
	m_gridmlp_loss_scale = gridmlp_loss_scale(n);
	check(ngp_hip_loss_and_gradient(m_stream, (int)m_nerf.training.loss_type, n, dims, m_gridmlp_loss_scale, m_gm_out.as<uint16_t>(), gm_out_stride(), targets, m_gm_values.as<float>(), m_dloss.as<uint16_t>(),
	                                gm_out_stride()), "loss_and_gradient");
	profile_begin(PK_BACKWARD);
	if (m_gated) {
		const uint32_t f = m_gated_block.n_hidden;
		uint16_t *const w = m_params.as<uint16_t>(), *const g = m_grads.as<uint16_t>();
		m_gated_dx.enlarge((size_t)n * 32 * 2);
		m_gated_ws.enlarge(std::max<uint64_t>(16, ngp_hip_gated_ffn_workspace_bytes(&m_gated_block, n, NGP_FFN_BACKWARD)));
		check(ngp_hip_gated_ffn_backward(m_stream, &m_gated_block, n, m_x_saved.as<uint16_t>(), 32, w, w + 32 * f, w + 64 * f, m_dloss.as<uint16_t>(), gm_out_stride(), m_gated_dx.as<uint16_t>(), 32, g,
		                                 g + 32 * f, g + 64 * f, m_gated_ws.data(), m_gated_ws.bytes()), "gated_ffn_backward");
		m_bwd_scratch.enlarge(ngp_hip_grid_gradient_scratch_bytes(n));
		// as ngp_hip_gridmlp_backward: the stratified image batch runs along x, SDF samples have no order
		check(ngp_hip_grid_gradient(m_stream, n_dims, desc, pos, n_dims, n, m_gated_dx.as<uint16_t>(), n_dims == 2, g + m_n_matrix_params, m_bwd_scratch.data(), m_bwd_scratch.bytes()), "grid_gradient");
	} else
	check(ngp_hip_gridmlp_backward(m_stream, n_dims, desc, m_params.as<uint16_t>(), pos, n_dims, n, m_x_saved.as<uint16_t>(), m_dloss.as<uint16_t>(), gm_out_stride(), m_grads.as<uint16_t>(),
	                               m_bwd_scratch.data(), m_bwd_scratch.bytes()), "gridmlp_backward");
	profile_end(PK_BACKWARD, n);
	if (get_loss_scalar) {
		check(ngp_hip_reduce_sum_f32(m_stream, m_gm_values.as<float>(), n * dims, m_loss_scalar_gpu.as<float>()), "reduce_sum");
		sync();
		m_loss_scalar_gpu.copy_to_host(&m_loss_scalar, 4);
	}
	optimizer_step(m_gridmlp_loss_scale);
	++m_training_step;
}

// ---- P1: image ------------------------------------------------------------------------------------------------------------------------
void Testbed::load_image(const std::string& path) {  // Testbed::load_image (testbed_image.cu:362-434): .exr -> float RGBA, .bin -> half RGBA, else the 8-bit decoders
	auto ends_with = [&](const char* ext) { const size_t n = strlen(ext); if (path.size() < n) return false; std::string tail = path.substr(path.size() - n); std::transform(tail.begin(), tail.end(), tail.begin(), ::tolower); return tail == ext; };
	if (ends_with(".exr")) {   // load_exr_image (385-397)
		int w = 0, h = 0; std::vector<float> px;
		read_exr_rgba_f32(path, w, h, px);
		set_image_data(w, h, px.data());
		m_data_path = path;
		return;
	}
	if (!ends_with(".bin")) {  // load_stbi_image (399-412): load_stbi hands back linear premultiplied floats (tinyexr_wrapper.cu load_stbi: srgb_to_linear on rgb, alpha / 255)
		int w = 0, h = 0; std::vector<uint8_t> px8;
		read_image_rgba8(path, w, h, px8);
		std::vector<float> px((size_t)w * h * 4);
		for (size_t i = 0; i < (size_t)w * h; ++i) {
			const float a = (float)px8[i * 4 + 3] * (1.0f / 255.0f);
			for (int c = 0; c < 3; ++c) {
				const float v = (float)px8[i * 4 + c] * (1.0f / 255.0f);
				px[i * 4 + c] = (v <= 0.04045f ? v / 12.92f : std::pow((v + 0.055f) / 1.055f, 2.4f)) * a;
			}
			px[i * 4 + 3] = a;
		}
		set_image_data(w, h, px.data());
		m_data_path = path;
		return;
	}
	FILE* f = fopen(path.c_str(), "rb");
	if (!f) throw std::runtime_error{path + " does not exist."};
	int32_t hw[2];
	if (fread(hw, 4, 2, f) != 2 || hw[0] <= 0 || hw[1] <= 0) { fclose(f); throw std::runtime_error{"bad .bin image header in " + path}; }
	const size_t n_pixels = (size_t)hw[0] * hw[1];
	std::vector<uint16_t> px(n_pixels * 4);
	const size_t got = fread(px.data(), 2, px.size(), f);
	fclose(f);
	if (got != px.size()) throw std::runtime_error{"truncated .bin image " + path};
	m_image.resolution[1] = hw[0]; m_image.resolution[0] = hw[1];
	m_image.data.resize(px.size() * 2);
	m_image.data.copy_from_host(px.data(), px.size() * 2);
	m_image.type = 2;
	m_data_path = path;
	m_training_data_available = true;
}

void Testbed::set_image_data(int w, int h, const float* rgba_host) {
	if (m_testbed_mode != ETestbedMode::Image) throw std::runtime_error{"set_image_data: TestbedMode.Image only"};
	m_image.resolution[0] = w; m_image.resolution[1] = h;
	m_image.data.resize((size_t)w * h * 16);
	m_image.data.copy_from_host(rgba_host, (size_t)w * h * 16);
	m_image.type = 3;
	m_training_data_available = true;
}

void Testbed::train_image(uint32_t batch_size, bool get_loss_scalar) {  // testbed_image.cu:220-291
	const uint32_t n = batch_size;
	m_image.positions.enlarge((size_t)n * 8); m_image.targets.enlarge((size_t)n * 12);
	// generate_random_uniform<float>(stream, m_rng, n * 2, positions) [tcnn], then stratification when the batch is a square power of two (236-247)
	check(ngp_hip_generate_random_uniform(m_stream, m_rng.state, m_rng.inc, n * 2, m_image.positions.as<float>()), "generate_random_uniform");
	m_rng.advance((int64_t)n * 2);
	if (m_image.stratified) {
		uint32_t log2_batch = 0;
		while ((1u << log2_batch) < n) ++log2_batch;
		if ((1u << log2_batch) == n && log2_batch % 2 == 0) check(ngp_hip_image_stratify2(m_stream, n, log2_batch, m_image.positions.as<float>()), "stratify2");
	}
	check(ngp_hip_image_eval_and_snap(m_stream, n, m_image.data.data(), m_image.type, m_image.positions.as<float>(), m_image.resolution, m_image.targets.as<float>(), 3,
	                                  m_image.snap_to_pixel_centers, m_image.linear_colors), "eval_image_and_snap");
	gridmlp_training_step(m_image.positions.as<float>(), 2, m_image.targets.as<float>(), 3, n, get_loss_scalar);
}

void Testbed::render_image(RenderBuffer& rb) {  // testbed_image.cu:293-360 (no activation visualisation)
	const uint32_t n_pixels = (uint32_t)rb.res[0] * (uint32_t)rb.res[1];
	const uint32_t n_elements = next_multiple(n_pixels, BATCH_SIZE_GRANULARITY);
	m_image.render_coords.enlarge((size_t)n_elements * 8); m_image.render_out.enlarge((size_t)n_elements * gm_out_stride() * 2);
	const float sc[2] = {m_screen_center[0] - 0.5f, m_screen_center[1] - 0.5f};
	HIP_TRY(hipMemsetAsync(m_image.render_coords.data(), 0, (size_t)n_elements * 8, (hipStream_t)m_stream));
	check(ngp_hip_image_init_coords(m_stream, m_image.render_coords.as<float>(), rb.res, m_image.resolution, m_scale, m_image.pos, sc, m_snap_to_pixel_centers, rb.spp), "image_init_coords");
	join_side_ema();
	gridmlp_inference(m_inference_params.as<uint16_t>(), m_image.render_coords.as<float>(), 2, n_elements, m_image.render_out.as<uint16_t>(), "gridmlp_forward (render)");
	check(ngp_hip_image_shade(m_stream, rb.res, m_image.render_coords.as<float>(), m_image.render_out.as<uint16_t>(), gm_out_stride(), rb.frame_buffer.as<float>(), rb.depth_buffer.as<float>(),
	                          m_image.linear_colors), "image_shade");
}

float Testbed::compute_image_mse(bool quantize_to_byte) {  // testbed_image.cu:461-523
	if (m_testbed_mode != ETestbedMode::Image || m_n_params == 0 || !m_image.type) throw std::runtime_error{"compute_image_mse: needs Image mode with an image and a network"};
	const uint32_t n_elements = (uint32_t)m_image.resolution[0] * (uint32_t)m_image.resolution[1];
	const uint32_t max_batch = 1u << 20;
	m_image.se.enlarge((size_t)(n_elements + 256) * 4);
	DeviceBuffer pos, targets, pred;
	pos.resize((size_t)max_batch * 8); targets.resize((size_t)max_batch * 12); pred.resize((size_t)max_batch * gm_out_stride() * 2);
	for (uint32_t offset = 0; offset < n_elements; offset += max_batch) {
		const uint32_t count = std::min(max_batch, n_elements - offset);
		const uint32_t batch = (count + 255u) & ~255u;
		check(ngp_hip_image_coords_from_idx(m_stream, batch, offset, pos.as<float>(), m_image.resolution), "image_coords_from_idx");
		check(ngp_hip_image_eval_and_snap(m_stream, batch, m_image.data.data(), m_image.type, pos.as<float>(), m_image.resolution, targets.as<float>(), 3, 1, m_image.linear_colors), "eval_image_and_snap");
		join_side_ema();
		gridmlp_inference(m_inference_params.as<uint16_t>(), pos.as<float>(), 2, batch, pred.as<uint16_t>(), "gridmlp_forward (mse)");
		check(ngp_hip_image_mse(m_stream, count, targets.as<float>(), pred.as<uint16_t>(), gm_out_stride(), m_image.se.as<float>() + offset, quantize_to_byte), "image_mse");
	}
	check(ngp_hip_reduce_sum_f32(m_stream, m_image.se.as<float>(), n_elements, m_loss_scalar_gpu.as<float>()), "reduce_sum");
	sync();
	float sum = 0.f;
	m_loss_scalar_gpu.copy_to_host(&sum, 4);
	return sum / (float)n_elements;
}

// ---- P2: sdf (training step on provided samples) --------------------------------------------------------------------------------------------
void Testbed::override_sdf_training_data(const float* points, const float* distances, size_t n) {  // python_api.cu:74-100
	if (m_testbed_mode != ETestbedMode::Sdf) throw std::runtime_error{"override_sdf_training_data: TestbedMode.Sdf only"};
	if (n == 0) throw std::runtime_error{"Invalid Points<->Distances data"};
	// the reference maps the points into the unit cube of the loaded mesh (raw_aabb, mesh_scale); without a mesh the caller provides unit-cube data
	m_sdf.positions.resize(n * 12); m_sdf.distances.resize(n * 4);
	m_sdf.positions.copy_from_host(points, n * 12);
	m_sdf.distances.copy_from_host(distances, n * 4);
	m_sdf.n_samples = (uint32_t)n; m_sdf.cursor = 0;
	m_training_data_available = true;
}

void Testbed::train_sdf(uint32_t batch_size, bool get_loss_scalar) {  // testbed_sdf.cu:1229-1252
	if (m_sdf.n_samples < batch_size) throw std::runtime_error{"train(): fewer SDF samples provided than the batch size"};
	if (m_sdf.cursor + batch_size > m_sdf.n_samples) m_sdf.cursor = 0;   // walk the provided set batch by batch
	const float* pos = m_sdf.positions.as<float>() + (size_t)m_sdf.cursor * 3;
	const float* dist = m_sdf.distances.as<float>() + m_sdf.cursor;
	m_sdf.cursor += batch_size;
	gridmlp_training_step(pos, 3, dist, 1, batch_size, get_loss_scalar);
}

} // namespace ngp
